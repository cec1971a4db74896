/*
 * gact._fused: the host side of gact.fused (argument checks, allocation, library calls) as native code.
 *
 * The operators are called once or twice per layer and step, several of them in front of kernels of a few microseconds;
 * written in Python their checks, allocations and ctypes calls cost 20 us per call, here about 5.  Like gact._hooks this
 * module belongs to the Python layer (it links against libtorch) and reaches the kernels through the C ABI of
 * libgact_b200.so.  Errors are raised as Python exceptions: RuntimeError for tensors the operators cannot take (device,
 * type), ValueError for shapes, TypeError for wrong kinds of arguments.
 */
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <vector>

#include "gact_b200.h"

namespace {

using at::Tensor;

long long g_launches = 0;          // library kernels enqueued from here

int type_code(at::ScalarType t) {
    switch (t) {
    case at::kFloat: return GACT_F32;
    case at::kHalf: return GACT_F16;
    case at::kBFloat16: return GACT_BF16;
    default: return -1;
    }
}

void check(int status, const char* what) {
    if (status == GACT_OK) return;
    const std::string msg = std::string(what) + ": " + gact_error_string(status) + " (status " + std::to_string(status) + ")";
    if (status == GACT_ERR_SIZE || status == GACT_ERR_DTYPE || status == GACT_ERR_MODE) C10_THROW_ERROR(ValueError, msg);
    C10_THROW_ERROR(Error, msg);
}

// An earlier call's copy that never arrived left its results incomplete: said by the next call, whoever made the first one.
void check_reports() {
    TORCH_CHECK(gact_pipeline_reported() == 0, "gact.fused: a copy of a product or of layer norm's rows did not arrive within its wait limit; results "
                "of calls since the last check are incomplete");
}

void check_tensor(const Tensor& t, const char* name, bool half_only, const Tensor* like) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor!");
    TORCH_CHECK(t.layout() == at::kStrided, name, " must be a dense tensor");
    const int c = type_code(t.scalar_type());
    TORCH_CHECK(c >= 0 && !(half_only && c == GACT_F32), "The type of ", name, " is not correct!");
    if (like) TORCH_CHECK(t.device() == like->device(), name, " is on ", t.device().str(), ", the input on ", like->device().str());
}

int64_t rows_of(const Tensor& t) {
    int64_t n = 1;
    for (int64_t i = 0; i + 1 < t.dim(); i++) n *= t.size(i);
    return n;
}

// t as rows of its last dimension with unit stride inside a row; copies only what cannot be described that way
struct Rows { Tensor t; int64_t rows, ld; };
Rows as_rows(const Tensor& t) {
    const int64_t cols = t.size(-1), rows = rows_of(t);
    if (t.is_contiguous()) return {t, rows, cols};
    Tensor u = t.dim() == 2 ? t : t.reshape({rows, cols});
    if (cols > 1 && u.stride(1) != 1) u = u.contiguous();
    int64_t ld = rows > 1 ? u.stride(0) : cols;
    if (ld < cols) {                                 // expanded rows
        u = u.contiguous();
        ld = cols;
    }
    return {u, rows, ld};
}

// uninitialised memory of the caching allocator, without the dispatcher's detour
Tensor make(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
    return Tensor(at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt));
}

// an operand that a tensor map can describe: base and pitch multiples of 16 bytes; anything else is copied to such a pitch
Rows as_operand(Rows r, int64_t cols, void* stream) {
    if (r.ld % 8 == 0 && ((uintptr_t)r.t.data_ptr() & 15) == 0) return r;
    const int64_t pitch = (cols + 7) / 8 * 8;
    Tensor out = make({r.rows, pitch}, r.t.scalar_type(), r.t);
    check(gact_repitch16(r.t.data_ptr(), r.ld, r.rows, cols, out.data_ptr(), pitch, stream), "gact_repitch16");
    g_launches++;
    return {out, r.rows, pitch};
}

// how codes are rounded; `held` keeps a seed that lies on the device
struct Seed { int rounding = 0; uint64_t value = 0; Tensor held; };

// A checkpoint is one byte tensor: rows x pitch codes, then rows x pitch / 32 scales.
struct Codes {
    Tensor buf; int64_t split = 0;
    bool defined() const { return buf.defined(); }
    void* codes() const { return buf.defined() ? buf.data_ptr() : nullptr; }
    void* scales() const { return buf.defined() ? (char*)buf.data_ptr() + split : nullptr; }
};
Codes empty_codes(int64_t rows, int64_t cols, const Tensor& like) {
    const int64_t n = rows * gact_checkpoint8_pitch(cols);
    return {make({n + n / GACT_BLOCK8}, at::kChar, like), n};
}
// `buf` as the checkpoint of rows x cols
Codes as_codes(const Tensor& buf, int64_t rows, int64_t cols, const Tensor* like) {
    const int64_t n = rows * gact_checkpoint8_pitch(cols);
    TORCH_CHECK(buf.is_cuda(), "checkpoint must be a CUDA tensor!");
    TORCH_CHECK_VALUE(buf.dim() == 1 && buf.scalar_type() == at::kChar && buf.is_contiguous() && buf.size(0) == n + n / GACT_BLOCK8,
                      "the checkpoint of ", rows, " x ", cols, " elements takes ", n + n / GACT_BLOCK8, " contiguous int8, got ", buf.sizes());
    if (like) TORCH_CHECK(buf.device() == like->device(), "checkpoint is on ", buf.device().str(), ", the input on ", like->device().str());
    return {buf, n};
}
bool is_codes(const Tensor& t) { return t.defined() && t.scalar_type() == at::kChar; }

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream_of(const Tensor& t) { return (void*)c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
Tensor scratch(int64_t bytes, const Tensor& like) { return bytes > 0 ? make({bytes}, at::kByte, like) : Tensor(); }
std::vector<int64_t> with_last(const Tensor& t, int64_t last) {
    std::vector<int64_t> s = t.sizes().vec();
    s.back() = last;
    return s;
}

Codes checkpoint8(const Tensor& x, const Seed& seed) {
    const Rows r = as_rows(x);
    const int64_t cols = x.size(-1);
    Codes c = empty_codes(r.rows, cols, x);
    if (x.numel() == 0) return c;
    check(gact_checkpoint8(r.t.data_ptr(), type_code(x.scalar_type()), r.rows, cols, r.ld, seed.rounding, seed.value, c.codes(), c.scales(),
                           stream_of(x)), "gact_checkpoint8");
    g_launches++;
    return c;
}

// ---- argument conversion ----------------------------------------------------------------------------------------------
Tensor tensor_arg(PyObject* o, const char* name) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
    return THPVariable_Unpack(o);
}
Tensor optional_arg(PyObject* o, const char* name) { return o == Py_None ? Tensor() : tensor_arg(o, name); }
// None, a number, or a tensor beside `like` whose one int64 the kernels read
Seed seed_arg(PyObject* o, const Tensor& like) {
    Seed s;
    if (THPVariable_Check(o)) {
        s.held = THPVariable_Unpack(o);
        TORCH_CHECK(s.held.device() == like.device(), "seed is on ", s.held.device().str(), ", the input on ", like.device().str());
        TORCH_CHECK_VALUE(s.held.scalar_type() == at::kLong && s.held.numel() == 1 && s.held.layout() == at::kStrided, "a seed tensor holds one int64");
        s.rounding = GACT_CODES_STOCHASTIC | GACT_CODES_DEVICE_SEED;
        s.value = (uint64_t)(uintptr_t)s.held.data_ptr();
    } else if (o != Py_None) {
        s.rounding = GACT_CODES_STOCHASTIC;
        s.value = PyLong_AsUnsignedLongLongMask(o);
        if (PyErr_Occurred()) throw python_error();
    }
    return s;
}
bool bool_arg(PyObject* o) {
    const int t = PyObject_IsTrue(o);
    if (t < 0) throw python_error();
    return t != 0;
}
PyObject* wrap(const Tensor& t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}
PyObject* tuple_of(std::initializer_list<Tensor> ts) {
    PyObject* out = PyTuple_New((Py_ssize_t)ts.size());
    if (!out) throw python_error();
    Py_ssize_t i = 0;
    for (const Tensor& t : ts) PyTuple_SET_ITEM(out, i++, wrap(t));
    return out;
}
void count_args(Py_ssize_t n, Py_ssize_t want) { TORCH_CHECK_TYPE(n == want, "takes ", want, " arguments, got ", n); }
// what every entry point begins with
void enter(Py_ssize_t n, Py_ssize_t want) {
    count_args(n, want);
    check_reports();
}

// ---- entry points -----------------------------------------------------------------------------------------------------
// checkpoint8(input, seed) -> buffer
PyObject* py_checkpoint8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    enter(nargs, 2);
    const Tensor x = tensor_arg(args[0], "input");
    check_tensor(x, "input", false, nullptr);
    TORCH_CHECK_VALUE(x.dim() > 0, "input needs at least one dimension");
    at::AutoDispatchBelowADInplaceOrView below;
    c10::cuda::CUDAGuard guard(x.device());
    return wrap(checkpoint8(x, seed_arg(args[1], x)).buf);
    END_HANDLE_TH_ERRORS
}

// restore8(buffer, shape, dtype) -> tensor
PyObject* py_restore8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    enter(nargs, 3);
    const Tensor buf = tensor_arg(args[0], "checkpoint");
    TORCH_CHECK_TYPE(PyTuple_Check(args[1]), "shape must be a tuple");
    TORCH_CHECK_TYPE(THPDtype_Check(args[2]), "dtype must be a torch.dtype");
    std::vector<int64_t> shape;
    int64_t rows = 1;
    const Py_ssize_t nd = PyTuple_GET_SIZE(args[1]);
    for (Py_ssize_t i = 0; i < nd; i++) {
        shape.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(args[1], i)));
        if (PyErr_Occurred()) throw python_error();
        if (i + 1 < nd) rows *= shape.back();
    }
    const at::ScalarType st = reinterpret_cast<THPDtype*>(args[2])->scalar_type;
    TORCH_CHECK(type_code(st) >= 0, "The type of the result is not correct!");
    TORCH_CHECK_VALUE(nd > 0, "a checkpoint has at least one dimension");
    const Codes c = as_codes(buf, rows, shape.back(), nullptr);
    at::AutoDispatchBelowADInplaceOrView below;
    c10::cuda::CUDAGuard guard(buf.device());
    const Tensor out = make(shape, st, buf);
    if (out.numel() > 0) {
        check(gact_restore8(c.codes(), c.scales(), rows, shape.back(), type_code(st), out.data_ptr(), shape.back(), stream_of(out)),
              "gact_restore8");
        g_launches++;
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// type of weight and bias (that of the input, or fp32; both alike)
at::ScalarType param_type(const Tensor& w, const Tensor& b, int64_t cols, const Tensor& x) {
    at::ScalarType t = x.scalar_type();
    bool seen = false;
    const Tensor* ps[2] = {&w, &b};
    for (int i = 0; i < 2; i++) {
        const Tensor& p = *ps[i];
        const char* name = i ? "bias" : "weight";
        if (!p.defined()) continue;
        check_tensor(p, name, false, &x);
        TORCH_CHECK_VALUE(p.dim() == 1 && p.size(0) == cols, name, " must have shape (", cols, ",)");
        TORCH_CHECK((p.scalar_type() == x.scalar_type() || p.scalar_type() == at::kFloat) && (!seen || p.scalar_type() == t), "The type of ", name,
                    " is not correct!");
        t = p.scalar_type();
        seen = true;
    }
    return t;
}

// layer_norm(input, weight, bias, eps, compress, seed, save, center) -> (y, checkpoint or input, statistics, weight)
PyObject* py_layer_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    enter(nargs, 8);
    const Tensor x = tensor_arg(args[0], "input");
    Tensor w = optional_arg(args[1], "weight"), b = optional_arg(args[2], "bias");
    const double eps = PyFloat_AsDouble(args[3]);
    if (PyErr_Occurred()) throw python_error();
    const bool compress = bool_arg(args[4]), save = bool_arg(args[6]), center = bool_arg(args[7]);
    check_tensor(x, "input", false, nullptr);
    const Seed seed = seed_arg(args[5], x);
    TORCH_CHECK_VALUE(x.dim() > 0, "input needs at least one dimension");
    const int64_t cols = x.size(-1);
    TORCH_CHECK_VALUE(cols >= 1 && cols <= GACT_LAYER_NORM_MAX_COLS, "layer norm takes rows of 1 to ", GACT_LAYER_NORM_MAX_COLS, " elements, got ", cols);
    const at::ScalarType pt = param_type(w, b, cols, x);
    at::AutoDispatchBelowADInplaceOrView below;
    c10::cuda::CUDAGuard guard(x.device());
    if (w.defined()) w = w.contiguous();
    if (b.defined()) b = b.contiguous();
    const Rows r = as_rows(x);
    const Tensor y = make(x.sizes(), x.scalar_type(), x);
    Codes c;
    Tensor stats;
    if (save) {
        stats = make({r.rows, 2}, at::kFloat, x);
        if (compress) c = empty_codes(r.rows, cols, x);
    }
    if (r.rows > 0) {
        check(gact_layer_norm(r.t.data_ptr(), type_code(x.scalar_type()), r.rows, cols, r.ld, ptr(w), ptr(b), type_code(pt), eps, y.data_ptr(),
                              (float*)ptr(stats), c.codes(), c.scales(),
                              seed.rounding | (center ? GACT_CODES_CENTERED : 0), seed.value, stream_of(x)),
              "gact_layer_norm");
        g_launches++;
    }
    return tuple_of({y, !save ? Tensor() : compress ? c.buf : x, stats, w});
    END_HANDLE_TH_ERRORS
}

// layer_norm_backward(grad_output, checkpoint or input, statistics, weight, fp32 parameters, need_input, need_weight,
//                     need_bias) -> (grad of the input, of weight, of bias)
PyObject* py_layer_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    enter(nargs, 8);
    const Tensor dy = tensor_arg(args[0], "grad_output"), kept = tensor_arg(args[1], "saved input"), stats = tensor_arg(args[2], "saved statistics"),
                 w = optional_arg(args[3], "weight");
    const bool f32 = bool_arg(args[4]), nx = bool_arg(args[5]), nw = bool_arg(args[6]), nb = bool_arg(args[7]);
    check_tensor(dy, "grad_output", false, &stats);
    TORCH_CHECK_VALUE(dy.dim() > 0, "grad_output needs at least one dimension");
    at::AutoDispatchBelowADInplaceOrView below;
    c10::cuda::CUDAGuard guard(dy.device());
    const int64_t cols = dy.size(-1);
    const Rows r = as_rows(dy);
    TORCH_CHECK_VALUE(stats.dim() == 2 && stats.size(0) == r.rows && stats.size(1) == 2 && stats.is_contiguous() && stats.scalar_type() == at::kFloat,
                      "saved statistics do not fit grad_output");
    Rows x{Tensor(), 0, 0};
    Codes c;
    if (is_codes(kept)) {
        c = as_codes(kept, r.rows, cols, &dy);
    } else {
        check_tensor(kept, "saved input", false, &dy);
        TORCH_CHECK_VALUE(kept.sizes() == dy.sizes() && kept.scalar_type() == dy.scalar_type(), "saved input does not fit grad_output");
        x = as_rows(kept);
    }
    const at::ScalarType pt = f32 ? at::kFloat : dy.scalar_type();
    if (w.defined()) {
        check_tensor(w, "weight", false, &dy);
        TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == cols && w.is_contiguous() && w.scalar_type() == pt, "weight does not fit grad_output");
    }
    Tensor dx, dw, db, scr;
    if (nx) dx = make(dy.sizes(), dy.scalar_type(), dy);
    if (nw) dw = make({cols}, pt, dy);
    if (nb) db = make({cols}, pt, dy);
    if (nw || nb) scr = scratch(gact_layer_norm_backward_scratch_bytes(r.rows, cols), dy);
    if (nx || nw || nb) {
        check(gact_layer_norm_backward(r.t.data_ptr(), type_code(dy.scalar_type()), r.rows, cols, r.ld, ptr(x.t), x.ld, c.codes(), c.scales(),
                                       (const float*)stats.data_ptr(), ptr(w), type_code(pt), ptr(dx), ptr(dw), ptr(db), ptr(scr), stream_of(dy)),
              "gact_layer_norm_backward");
        g_launches += 1 + (nw || nb);
    }
    return tuple_of({dx, dw, db});
    END_HANDLE_TH_ERRORS
}

// linear(input, weight, bias, activation code, residual, compress, seed, save, checkpoint of the input or None, keep input)
//   -> (y, checkpoint or input, checkpoint of z or z)
PyObject* py_linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    enter(nargs, 10);
    const Tensor x = tensor_arg(args[0], "input"), w = tensor_arg(args[1], "weight");
    Tensor b = optional_arg(args[2], "bias");
    const int act = (int)PyLong_AsLong(args[3]);
    if (PyErr_Occurred()) throw python_error();
    const Tensor res = optional_arg(args[4], "residual");
    const bool compress = bool_arg(args[5]), save = bool_arg(args[7]), keep = save && bool_arg(args[9]);
    const Tensor given = optional_arg(args[8], "checkpoint");
    check_tensor(x, "input", true, nullptr);
    const Seed seed = seed_arg(args[6], x);
    check_tensor(w, "weight", true, &x);
    TORCH_CHECK(w.scalar_type() == x.scalar_type(), "The type of weight is not correct!");
    TORCH_CHECK_VALUE(x.dim() > 0 && w.dim() == 2 && x.size(-1) == w.size(1), "input ", x.sizes(), " does not fit weight ", w.sizes());
    const int64_t cout = w.size(0), cin = w.size(1);
    TORCH_CHECK_VALUE(cin > 0 && cout > 0, "a linear layer needs at least one input and one output feature");
    const std::vector<int64_t> out_shape = with_last(x, cout);
    if (b.defined()) {
        check_tensor(b, "bias", true, &x);
        TORCH_CHECK(b.scalar_type() == x.scalar_type(), "The type of bias is not correct!");
        TORCH_CHECK_VALUE(b.dim() == 1 && b.size(0) == cout, "bias must have shape (", cout, ",)");
    }
    if (res.defined()) {
        check_tensor(res, "residual", true, &x);
        TORCH_CHECK(res.scalar_type() == x.scalar_type(), "The type of residual is not correct!");
        TORCH_CHECK_VALUE(res.sizes() == at::IntArrayRef(out_shape), "residual must have shape ", at::IntArrayRef(out_shape), ", got ", res.sizes());
    }
    at::AutoDispatchBelowADInplaceOrView below;
    c10::cuda::CUDAGuard guard(x.device());
    if (b.defined()) b = b.contiguous();
    Rows xr = as_rows(x), wr = as_rows(w);
    Rows rr{Tensor(), 0, 0};
    if (res.defined()) rr = as_rows(res);
    Codes c;
    if (given.defined()) c = as_codes(given, xr.rows, cin, &x);
    const Tensor y = make(out_shape, x.scalar_type(), x);
    Codes zc, xc;                                        // xc: the checkpoint of x that this call makes
    Tensor z;
    if (save) {
        if (act && compress) zc = empty_codes(xr.rows, cout, x);
        else if (act) z = make({xr.rows, cout}, x.scalar_type(), x);
        if (keep && compress && !c.defined()) c = xc = empty_codes(xr.rows, cin, x);
    }
    if (xr.rows > 0) {
        void* s = stream_of(x);
        xr = as_operand(xr, cin, s);
        wr = as_operand(wr, cin, s);
        const int64_t bytes = gact_linear_scratch_bytes(xr.rows, cin, cout, 0);
        const Tensor scr = scratch(bytes, x);
        check(gact_linear(xr.t.data_ptr(), xr.ld, wr.t.data_ptr(), wr.ld, ptr(b), ptr(rr.t), rr.ld, type_code(x.scalar_type()), xr.rows, cin, cout, act,
                          y.data_ptr(), xc.codes(), xc.scales(), ptr(z), zc.codes(), zc.scales(), seed.rounding, seed.value, ptr(scr), s),
              "gact_linear");
        g_launches += 1 + (bytes > 0);
    }
    if (!save) return tuple_of({y, Tensor(), Tensor()});
    return tuple_of({y, !keep ? Tensor() : compress ? c.buf : x, zc.defined() ? zc.buf : z});
    END_HANDLE_TH_ERRORS
}

// linear_backward(grad_output, weight or None, activation code, checkpoint or input or None, checkpoint of z or z or None,
//                 need_input, need_weight, need_bias, input features) -> (grad of the input, of weight, of bias)
PyObject* py_linear_backward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    enter(nargs, 9);
    const Tensor dy = tensor_arg(args[0], "grad_output"), w = optional_arg(args[1], "weight");
    const int act = (int)PyLong_AsLong(args[2]);
    if (PyErr_Occurred()) throw python_error();
    const Tensor xk = optional_arg(args[3], "saved input"), zk = optional_arg(args[4], "saved pre-activation");
    const bool nx = bool_arg(args[5]), nw = bool_arg(args[6]), nb = bool_arg(args[7]);
    const int64_t cin = PyLong_AsLongLong(args[8]);
    if (PyErr_Occurred()) throw python_error();
    check_tensor(dy, "grad_output", true, nullptr);
    TORCH_CHECK_VALUE(dy.dim() > 0 && dy.size(-1) > 0 && cin > 0, "grad_output ", dy.sizes(), " is not that of a linear layer");
    const int64_t cout = dy.size(-1);
    if (w.defined()) {
        check_tensor(w, "weight", true, &dy);
        TORCH_CHECK(dy.scalar_type() == w.scalar_type(), "The type of grad_output is not correct!");
        TORCH_CHECK_VALUE(w.dim() == 2 && cout == w.size(0) && cin == w.size(1), "grad_output ", dy.sizes(), " does not fit weight ", w.sizes());
    }
    TORCH_CHECK_VALUE(w.defined() || !nx, "the weight was not saved");
    TORCH_CHECK_VALUE(xk.defined() || !nw, "the input was not saved");
    const int code = type_code(dy.scalar_type());
    at::AutoDispatchBelowADInplaceOrView below;
    c10::cuda::CUDAGuard guard(dy.device());
    Rows dz = as_rows(dy);
    const int64_t rows = dz.rows;
    Tensor dx, dw, db;
    if (nx) dx = make(with_last(dy, cin), dy.scalar_type(), dy);
    if (nw) dw = make({cout, cin}, dy.scalar_type(), dy);
    if (nb) db = make({cout}, dy.scalar_type(), dy);
    if (rows == 0) {
        if (nw) dw.zero_();
        if (nb) db.zero_();
        return tuple_of({dx, dw, db});
    }
    void* s = stream_of(dy);
    const int64_t xb = nx ? gact_linear_scratch_bytes(rows, cin, cout, 1) : 0, wb = nw ? gact_linear_scratch_bytes(rows, cin, cout, 2) : 0;
    const Tensor scr = scratch(std::max(xb, wb), dy);          // (the two products run one after the other on this stream)
    const Tensor sums = scratch(nb ? gact_act_backward_scratch_bytes(rows, cout) : 0, dy);
    // dz = dy act'(z) and the partial sums of the bias gradient; without an activation, dy itself if a product can read it
    const bool readable = dz.ld % 8 == 0 && ((uintptr_t)dz.t.data_ptr() & 15) == 0;
    const bool make_dz = (nx || nw) && (act || !readable);
    if (nb || make_dz) {
        Rows z{Tensor(), 0, 0};
        Codes zc;
        Tensor out;
        const int64_t pitch = (cout + 7) / 8 * 8;
        if (act) {
            TORCH_CHECK_VALUE(zk.defined(), "the pre-activation was not saved");
            if (is_codes(zk)) {
                zc = as_codes(zk, rows, cout, &dy);
            } else {
                check_tensor(zk, "saved pre-activation", true, &dy);
                TORCH_CHECK_VALUE(zk.dim() == 2 && zk.size(0) == rows && zk.size(1) == cout && zk.scalar_type() == dy.scalar_type(),
                                  "saved pre-activation does not fit grad_output");
                z = as_rows(zk);
            }
        }
        if (act || make_dz) out = make({rows, pitch}, dy.scalar_type(), dy);
        check(gact_act_backward(dz.t.data_ptr(), code, rows, cout, dz.ld, act, ptr(z.t), z.ld, zc.codes(), zc.scales(), ptr(out), pitch,
                                nx || nw ? nullptr : ptr(db), ptr(sums), s), "gact_act_backward");
        g_launches += 1 + !(nx || nw);
        if (out.defined()) dz = {out, rows, pitch};
    }
    Codes xc;
    Rows x{Tensor(), 0, 0};
    if (nw) {
        if (is_codes(xk)) {
            xc = as_codes(xk, rows, cin, &dy);
            const int64_t pitch = gact_checkpoint8_pitch(cin);
            x = {make({rows, pitch}, dy.scalar_type(), dy), rows, pitch};
        } else {
            check_tensor(xk, "saved input", true, &dy);
            TORCH_CHECK_VALUE(xk.dim() > 0 && xk.size(-1) == cin && rows_of(xk) == rows && xk.scalar_type() == dy.scalar_type(),
                              "saved input does not fit grad_output");
            x = as_operand(as_rows(xk), cin, s);
        }
    }
    // beside the data gradient: the bias gradient's sums, and x restored for the weight gradient; without it the weight
    // gradient takes the sums and x is restored on its own
    if (nx) {
        const Rows wr = as_operand(as_rows(w), cin, s);
        check(gact_linear_dgrad(dz.t.data_ptr(), dz.ld, wr.t.data_ptr(), wr.ld, code, rows, cin, cout, dx.data_ptr(), ptr(sums), ptr(db), xc.codes(),
                                xc.scales(), xc.defined() ? x.t.data_ptr() : nullptr, ptr(scr), s), "gact_linear_dgrad");
        g_launches += 1 + (xb > 0);
    } else if (xc.defined()) {
        check(gact_restore8(xc.codes(), xc.scales(), rows, cin, code, x.t.data_ptr(), x.ld, s), "gact_restore8");
        g_launches++;
    }
    if (nw) {
        check(gact_linear_wgrad(dz.t.data_ptr(), dz.ld, x.t.data_ptr(), x.ld, code, rows, cin, cout, dw.data_ptr(), nx ? nullptr : ptr(sums),
                                nx ? nullptr : ptr(db), ptr(scr), s), "gact_linear_wgrad");
        g_launches += 1 + (wb > 0);
    }
    return tuple_of({dx, dw, db});
    END_HANDLE_TH_ERRORS
}

PyObject* py_launches(PyObject*, PyObject*) { return PyLong_FromLongLong(g_launches); }

#define FAST(f) (PyCFunction)(void (*)(void))f, METH_FASTCALL
PyMethodDef kMethods[] = {
    {"checkpoint8", FAST(py_checkpoint8), "checkpoint8(input, seed) -> buffer"},
    {"restore8", FAST(py_restore8), "restore8(buffer, shape, dtype) -> tensor"},
    {"layer_norm", FAST(py_layer_norm), "layer_norm(input, weight, bias, eps, compress, seed, save, center) -> (y, kept, statistics, weight)"},
    {"layer_norm_backward", FAST(py_layer_norm_backward),
     "layer_norm_backward(grad_output, kept, statistics, weight, fp32 parameters, need_input, need_weight, need_bias) -> three gradients"},
    {"linear", FAST(py_linear), "linear(input, weight, bias, activation, residual, compress, seed, save, checkpoint, keep_input) -> (y, kept, z)"},
    {"linear_backward", FAST(py_linear_backward),
     "linear_backward(grad_output, weight, activation, kept, z, need_input, need_weight, need_bias, input features) -> three gradients"},
    {"launches", py_launches, METH_NOARGS, "library kernels enqueued by this module"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fused", "Host side of gact.fused.", -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fused(void) { return PyModule_Create(&kModule); }
