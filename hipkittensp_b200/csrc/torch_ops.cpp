// Python extension `_torch_ops`: the tensor-level side of the operators that are called often and on little work (quantise,
// dequantise, the products, the layer norm): argument checks, result allocation, torch's current stream, and one call of the C ABI.
// gemm.py and norm.py hold the signatures and the documentation.  A call of the norm through ctypes and torch's Python
// allocators cost 12.6 us on the host, 3.7 of them in the C entry.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <optional>
#include <stdexcept>
#include <string>

#include "mxfp6.h"

namespace py = pybind11;

namespace {

// The entry points of the library instance the package has loaded (it may be another build than the one next to this file).
#define MX_ENTRIES(X) X(mxfp6_last_error) X(mxfp6_gemm_ex) X(mxfp6_gemm_ws) X(mxfp6_gemm_scaled) X(mxfp6_gemm_scaled_ws) X(mxfp6_quantize) X(mxfp6_dequantize_ex) X(mxfp6_layer_norm) \
    X(mxfp6_layer_norm_quantize) X(mxfp6_layer_norm_backward) X(mxfp6_layer_norm_backward_workspace_bytes)
struct Library {
#define X(name) decltype(&::name) name = nullptr;
    MX_ENTRIES(X)
#undef X
} lib;

[[noreturn]] void refuse(const std::string& what) { throw std::runtime_error(what); }

bool is_fp8(int fmt) { return fmt == MXFP8_E4M3 || fmt == MXFP8_E5M2; }
int64_t row_bytes(int64_t K, int fmt) { return is_fp8(fmt) ? K : fmt == MXFP4_E2M1 ? K / 2 : K * 3 / 4; }

const at::Tensor& tensor_of(py::handle h) {
    if (!THPVariable_Check(h.ptr())) refuse("Expected a torch.Tensor");
    return THPVariable_Unpack(h.ptr());
}

const char* name_of(at::ScalarType t) { return t == at::kByte ? "torch.uint8" : t == at::kBFloat16 ? "torch.bfloat16" : "torch.float32"; }

// a contiguous CUDA matrix of one type
const at::Tensor& matrix(py::handle h, const char* name, at::ScalarType dtype) {
    const at::Tensor& t = tensor_of(h);
    if (!t.is_contiguous()) refuse("Tensor must be contiguous");
    if (!t.is_cuda()) refuse("Tensor must be on CUDA device");
    if (t.dim() > 4) refuse("Expected Tensor.ndim <= 4");
    if (t.scalar_type() != dtype) refuse(std::string(name) + " must be " + name_of(dtype) + ", got " + std::string(py::str(h.attr("dtype"))));
    if (t.dim() != 2) refuse(std::string(name) + " must be 2-D");
    return t;
}

// K of an operand [rows, bytes]
int64_t k_of(const at::Tensor& t, int fmt, const char* name) {
    const int64_t n = t.size(1);
    if (is_fp8(fmt)) return n;
    if (fmt == MXFP4_E2M1) return 2 * n;
    if (n % 3) refuse(std::string(name) + ".shape[1] must be 3K/4 bytes");
    return n / 3 * 4;
}

// a contiguous CUDA matrix of fp32 or bf16 rows; *code: 0 = fp32, 1 = bf16
const at::Tensor& rows_of(py::handle h, const char* name, int* code) {
    const at::Tensor& t = tensor_of(h);
    if (!t.is_contiguous()) refuse("Tensor must be contiguous");
    if (!t.is_cuda()) refuse("Tensor must be on CUDA device");
    const at::ScalarType d = t.scalar_type();
    if ((d != at::kFloat && d != at::kBFloat16) || t.dim() != 2) refuse(std::string(name) + " must be a 2-D fp32 or bf16 tensor");
    *code = d == at::kFloat ? 0 : 1;
    return t;
}

// an optional contiguous vector of n elements on like's device; null when None
const void* vector_of(py::handle h, const char* name, int64_t n, const at::Tensor& like, bool bf16_too, int* code) {
    if (h.is_none()) return nullptr;
    const at::Tensor& t = tensor_of(h);
    if (!t.is_contiguous()) refuse("Tensor must be contiguous");
    if (!t.is_cuda() || t.get_device() != like.get_device()) refuse("all tensors must be on the same device");
    const at::ScalarType d = t.scalar_type();
    if (d != at::kFloat && !(bf16_too && d == at::kBFloat16)) refuse(std::string(name) + (bf16_too ? " must be fp32 or bf16" : " must be torch.float32"));
    if (t.dim() != 1 || t.size(0) != n) refuse(std::string(name) + " must have " + std::to_string(n) + " elements");
    if (code) *code = d == at::kFloat ? 0 : 1;
    return t.const_data_ptr();
}

void same_device(const at::Tensor& a, std::initializer_list<const at::Tensor*> others) {
    for (const at::Tensor* t : others)
        if (t->get_device() != a.get_device()) refuse("all tensors must be on the same device");
}

at::Tensor empty(at::IntArrayRef size, at::ScalarType dtype, const at::Tensor& like) {
    return at::detail::empty_cuda(size, dtype, like.device(), std::nullopt);
}

py::object wrap(at::Tensor t) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(std::move(t))); }

// the package's exception for an error code of the C ABI
py::object* g_error = nullptr;
void check(int rc) {
    if (rc == MXFP6_OK) return;
    py::object e = (*g_error)(rc, std::string(lib.mxfp6_last_error()));
    PyErr_SetObject(g_error->ptr(), e.ptr());
    throw py::error_already_set();
}

// entry(stream) on torch's current stream of t's device, with that device current and without the interpreter lock: a call's allocations, which
// stand in its entry, and its launch may wait for the device (a full queue, memory that is freed to make room, the library's first
// scratch buffer), and what the device waits for may be a callback that needs the lock.  (Released once per call: 0.1 us.)
template <typename F>
void launch(const at::Tensor& t, F entry) {
    const c10::DeviceIndex dev = (c10::DeviceIndex)t.get_device();
    int rc;
    {
        py::gil_scoped_release unlocked;
        c10::cuda::CUDAGuard guard(dev);
        rc = entry((void*)c10::cuda::getCurrentCUDAStream(dev).stream());
    }
    check(rc);
}

// ---------------------------------------------------------------------------------- products
struct Operands {
    const at::Tensor &a, &sa, &b, &sb;
    int64_t M, N, K;
};
Operands operands(py::handle A, py::handle scale_A, py::handle B, py::handle scale_B, int fmt, int fmt_b) {
    const at::Tensor &a = matrix(A, "A", at::kByte), &b = matrix(B, "B", at::kByte), &sa = matrix(scale_A, "scale_A", at::kByte),
                     &sb = matrix(scale_B, "scale_B", at::kByte);
    Operands o{a, sa, b, sb, a.size(0), b.size(0), k_of(a, fmt, "A")};
    if (k_of(b, fmt_b, "B") != o.K) refuse("A and B disagree on K");
    if (o.K % 32 || sa.size(0) != o.M || sa.size(1) != o.K / 32 || sb.size(0) != o.N || sb.size(1) != o.K / 32) refuse("scales must be [rows, K/32]");
    same_device(a, {&b, &sa, &sb});
    return o;
}
// the matrix a caller gives for the result; undefined when None
at::Tensor given_result(const Operands& o, py::handle out) {
    if (out.is_none()) return {};
    const at::Tensor& c = matrix(out, "C", at::kBFloat16);
    if (c.size(0) != o.M || c.size(1) != o.N) refuse("C must be [" + std::to_string(o.M) + ", " + std::to_string(o.N) + "]");
    same_device(o.a, {&c});
    return c;
}

// a caller's workspace, or none
struct Workspace {
    bool own = true;             // the library's
    void* ptr = nullptr;
    size_t bytes = 0;
};
Workspace workspace_of(const Operands& o, py::handle workspace) {
    if (workspace.is_none()) return {};
    const at::Tensor& w = tensor_of(workspace);
    if (!w.is_contiguous()) refuse("Tensor must be contiguous");
    if (w.scalar_type() != at::kByte) refuse("workspace must be torch.uint8");
    if (!w.is_cuda() || w.get_device() != o.a.get_device()) refuse("all tensors must be on the same device");
    return {false, w.mutable_data_ptr(), (size_t)w.numel()};
}

py::object gemm(py::handle A, py::handle scale_A, py::handle B, py::handle scale_B, int fmt, int fmt_b, py::handle out, py::handle workspace) {
    // the checks of dispatch_micro, in its order and words
    const at::Tensor &a = matrix(A, "A", at::kByte), &b = matrix(B, "B", at::kByte);
    const at::Tensor* given = out.is_none() ? nullptr : &matrix(out, "C", at::kBFloat16);
    const at::Tensor &sa = matrix(scale_A, "scale_A", at::kByte), &sb = matrix(scale_B, "scale_B", at::kByte);
    const Operands o{a, sa, b, sb, a.size(0), given ? given->size(1) : b.size(0), k_of(a, fmt, "A")};
    if (o.K % 128) refuse("K must be a multiple of 128");
    if (given && given->size(0) != o.M) refuse("C.shape[0] must equal A.shape[0]");
    if (b.size(0) != o.N || k_of(b, fmt_b, "B") != o.K) refuse("B must be [N, 3K/4] (fp6), [N, K] (fp8) or [N, K/2] (fp4) with the K of A");
    if (sa.size(0) != o.M || sa.size(1) != o.K / 32 || sb.size(0) != o.N || sb.size(1) != o.K / 32) refuse("scales must be [rows, K/32]");
    same_device(a, {&b, &sa, &sb});
    if (given) same_device(a, {given});
    const Workspace ws = workspace_of(o, workspace);
    at::Tensor c = given ? *given : at::Tensor();
    launch(o.a, [&](void* st) {
        if (!c.defined()) c = empty({o.M, o.N}, at::kBFloat16, o.a);
        const void *a = o.a.const_data_ptr(), *sa = o.sa.const_data_ptr(), *b = o.b.const_data_ptr(), *sb = o.sb.const_data_ptr();
        return ws.own ? lib.mxfp6_gemm_ex(a, sa, b, sb, c.mutable_data_ptr(), o.M, o.N, o.K, fmt, fmt_b, 0, st)
                      : lib.mxfp6_gemm_ws(a, sa, b, sb, c.mutable_data_ptr(), o.M, o.N, o.K, fmt, fmt_b, ws.ptr, ws.bytes, st);
    });
    return out.is_none() ? wrap(std::move(c)) : py::reinterpret_borrow<py::object>(out);
}

py::object gemm_scaled(py::handle A, py::handle scale_A, py::handle B, py::handle scale_B, py::handle row_scale, py::handle col_scale, py::handle bias,
                       int fmt, int fmt_b, py::handle out, py::handle workspace) {
    const Operands o = operands(A, scale_A, B, scale_B, fmt, fmt_b);
    auto vec = [&](py::handle h, const char* name, int64_t n) -> const float* {
        if (h.is_none()) return nullptr;
        if (!THPVariable_Check(h.ptr())) refuse(std::string(name) + " must be a contiguous fp32 tensor");
        const at::Tensor& t = tensor_of(h);
        if (t.scalar_type() != at::kFloat || !t.is_contiguous()) refuse(std::string(name) + " must be a contiguous fp32 tensor");
        if (!t.is_cuda() || t.get_device() != o.a.get_device()) refuse("Tensor must be on CUDA device");
        if (t.numel() != n) refuse(std::string(name) + " must have " + std::to_string(n) + " elements, has " + std::to_string(t.numel()));
        return (const float*)t.const_data_ptr();
    };
    const float *r = vec(row_scale, "row_scale", o.M), *cs = vec(col_scale, "col_scale", o.N), *bs = vec(bias, "bias", o.N);
    const Workspace ws = workspace_of(o, workspace);
    at::Tensor c = given_result(o, out);
    launch(o.a, [&](void* st) {
        if (!c.defined()) c = empty({o.M, o.N}, at::kBFloat16, o.a);
        const void *a = o.a.const_data_ptr(), *sa = o.sa.const_data_ptr(), *b = o.b.const_data_ptr(), *sb = o.sb.const_data_ptr();
        return ws.own ? lib.mxfp6_gemm_scaled(a, sa, b, sb, c.mutable_data_ptr(), r, cs, bs, o.M, o.N, o.K, fmt, fmt_b, st)
                      : lib.mxfp6_gemm_scaled_ws(a, sa, b, sb, c.mutable_data_ptr(), r, cs, bs, o.M, o.N, o.K, fmt, fmt_b, ws.ptr, ws.bytes, st);
    });
    return out.is_none() ? wrap(std::move(c)) : py::reinterpret_borrow<py::object>(out);
}

// ---------------------------------------------------------------------------------- quantise, dequantise
py::tuple quantize(py::handle X, int fmt) {
    const at::Tensor& x = tensor_of(X);
    if (!x.is_cuda()) refuse("Tensor must be on CUDA device");
    if ((x.scalar_type() != at::kFloat && x.scalar_type() != at::kBFloat16) || x.dim() != 2 || !x.is_contiguous())
        refuse("quantize expects a contiguous 2-D fp32 or bf16 tensor");
    const int64_t rows = x.size(0), K = x.size(1);
    if (K % 32) refuse("K must be a multiple of 32");
    at::Tensor packed, scales;
    launch(x, [&](void* st) {
        packed = empty({rows, row_bytes(K, fmt)}, at::kByte, x);
        scales = empty({rows, K / 32}, at::kByte, x);
        return lib.mxfp6_quantize(x.const_data_ptr(), x.scalar_type() == at::kFloat ? 0 : 1, rows, K, fmt, packed.mutable_data_ptr(), scales.mutable_data_ptr(), st);
    });
    return py::make_tuple(wrap(std::move(packed)), wrap(std::move(scales)));
}

py::object dequantize(py::handle P, py::handle S, int fmt, bool bf16) {
    const at::Tensor &p = matrix(P, "packed", at::kByte), &s = matrix(S, "scales", at::kByte);
    const int64_t rows = p.size(0), K = k_of(p, fmt, "packed");
    if (K % 32 || s.size(0) != rows || s.size(1) != K / 32) refuse("scales must be [rows, K/32]");
    same_device(p, {&s});
    at::Tensor out;
    launch(p, [&](void* st) {
        out = empty({rows, K}, bf16 ? at::kBFloat16 : at::kFloat, p);
        return lib.mxfp6_dequantize_ex(p.const_data_ptr(), s.const_data_ptr(), rows, K, fmt, out.mutable_data_ptr(), bf16 ? 1 : 0, st);
    });
    return wrap(std::move(out));
}

// ---------------------------------------------------------------------------------- layer norm
struct Norm {
    const at::Tensor& x;
    int code, wcode;
    int64_t rows, H;
    const void *w, *b;
};
Norm norm_of(py::handle X, py::handle weight, py::handle bias) {
    int code = 0, wc = 0, bc = 0;
    const at::Tensor& x = rows_of(X, "x", &code);
    const int64_t H = x.size(1);
    if (H < 1) refuse("x must have at least one column");
    const void *w = vector_of(weight, "weight", H, x, true, &wc), *b = vector_of(bias, "bias", H, x, true, &bc);
    if (w && b && wc != bc) refuse("weight and bias must have the same dtype");
    return {x, code, w ? wc : bc, x.size(0), H, w, b};
}

py::tuple layer_norm(py::handle X, py::handle weight, py::handle bias, double eps, py::handle out) {
    const Norm n = norm_of(X, weight, bias);
    at::Tensor y;
    if (!out.is_none()) {
        int code = 0;
        y = rows_of(out, "out", &code);
        if (y.sizes() != n.x.sizes() || code != n.code || y.get_device() != n.x.get_device()) refuse("out must have the shape, dtype and device of x");
    }
    at::Tensor mean, rstd;
    launch(n.x, [&](void* st) {
        if (!y.defined()) y = empty({n.rows, n.H}, n.x.scalar_type(), n.x);
        mean = empty({n.rows}, at::kFloat, n.x);
        rstd = empty({n.rows}, at::kFloat, n.x);
        return lib.mxfp6_layer_norm(n.x.const_data_ptr(), n.code, n.w, n.b, n.wcode, y.mutable_data_ptr(), (float*)mean.mutable_data_ptr(),
                                (float*)rstd.mutable_data_ptr(), n.rows, n.H, (float)eps, st);
    });
    return py::make_tuple(out.is_none() ? wrap(std::move(y)) : py::reinterpret_borrow<py::object>(out), wrap(std::move(mean)), wrap(std::move(rstd)));
}

py::tuple layer_norm_quantize(py::handle X, py::handle weight, py::handle bias, double eps, int fmt) {
    const Norm n = norm_of(X, weight, bias);
    if (n.H % 32) refuse("H must be a multiple of 32");
    at::Tensor packed, scales, mean, rstd;
    launch(n.x, [&](void* st) {
        packed = empty({n.rows, row_bytes(n.H, fmt)}, at::kByte, n.x);
        scales = empty({n.rows, n.H / 32}, at::kByte, n.x);
        mean = empty({n.rows}, at::kFloat, n.x);
        rstd = empty({n.rows}, at::kFloat, n.x);
        return lib.mxfp6_layer_norm_quantize(n.x.const_data_ptr(), n.code, n.w, n.b, n.wcode, fmt, packed.mutable_data_ptr(), scales.mutable_data_ptr(),
                                         (float*)mean.mutable_data_ptr(), (float*)rstd.mutable_data_ptr(), n.rows, n.H, (float)eps, st);
    });
    return py::make_tuple(wrap(std::move(packed)), wrap(std::move(scales)), wrap(std::move(mean)), wrap(std::move(rstd)));
}

py::tuple layer_norm_backward(py::handle DY, py::handle X, py::handle mean, py::handle rstd, py::handle weight) {
    const Norm n = norm_of(X, weight, py::none());
    int code = 0;
    const at::Tensor& dy = rows_of(DY, "dy", &code);
    if (dy.sizes() != n.x.sizes() || code != n.code || dy.get_device() != n.x.get_device()) refuse("dy must have the shape, dtype and device of x");
    if (mean.is_none() || rstd.is_none()) refuse("Expected a torch.Tensor");
    const float *m = (const float*)vector_of(mean, "mean", n.rows, n.x, false, nullptr), *r = (const float*)vector_of(rstd, "rstd", n.rows, n.x, false, nullptr);
    at::Tensor dx, dw, db;
    launch(n.x, [&](void* st) {
        dx = empty({n.rows, n.H}, n.x.scalar_type(), n.x);
        dw = empty({n.H}, at::kFloat, n.x);
        db = empty({n.H}, at::kFloat, n.x);
        const size_t bytes = lib.mxfp6_layer_norm_backward_workspace_bytes(n.rows, n.H);
        at::Tensor work = empty({(int64_t)bytes}, at::kByte, n.x);
        return lib.mxfp6_layer_norm_backward(dy.const_data_ptr(), n.x.const_data_ptr(), n.code, m, r, n.w, n.wcode, dx.mutable_data_ptr(),
                                         (float*)dw.mutable_data_ptr(), (float*)db.mutable_data_ptr(), n.rows, n.H, work.mutable_data_ptr(), bytes, st);
    });
    return py::make_tuple(wrap(std::move(dx)), wrap(std::move(dw)), wrap(std::move(db)));
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
    m.doc() = "tensor-level entry points over libmxfp6 (see gemm.py and norm.py)";
    // errors of torch's allocator keep their Python types (torch.OutOfMemoryError among them)
    py::register_local_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const c10::Error&) {
            torch::translate_exception_to_python(p);
        }
    });
    m.def("bind", [](uintptr_t handle, py::object error_class) {
#define X(name)                                                                              \
        lib.name = reinterpret_cast<decltype(&::name)>(dlsym(reinterpret_cast<void*>(handle), #name)); \
        if (!lib.name) throw std::runtime_error("the library has no " #name);
        MX_ENTRIES(X)
#undef X
        g_error = new py::object(std::move(error_class));      // never destroyed: outlives interpreter shutdown order problems
    });
    m.def("gemm", &gemm);
    m.def("gemm_scaled", &gemm_scaled);
    m.def("quantize", &quantize);
    m.def("dequantize", &dequantize);
    m.def("layer_norm", &layer_norm);
    m.def("layer_norm_quantize", &layer_norm_quantize);
    m.def("layer_norm_backward", &layer_norm_backward);
}
