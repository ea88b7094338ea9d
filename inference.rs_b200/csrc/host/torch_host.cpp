// The torch front end's call path in native code: argument checks, output allocation, stream look-up and the C-ABI call of one
// operation, without the interpreter in between. A decode call's kernel runs 4-15 us; the same steps in Python (tensor
// attribute look-ups, torch.cuda.current_stream, ctypes argument conversion) took 17-20 us of the host per call, here about 4.
//
// The module calls the C ABI through addresses handed over by bind() (the library that kernel_library.py found and checked), so
// there is one place that decides which library is used. Anything out of the ordinary (a wrong type, shape or device) makes a
// function return None instead of launching: the Python caller then takes its own path, which raises the proper error.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/_to_copy.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>  // C++ exceptions become the Python ones torch raises itself (OutOfMemoryError among them)
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <initializer_list>

namespace {

using at::Tensor;
using c10::ScalarType;

enum { TYPE_Q8_0 = 8, TYPE_Q4_K = 12, TYPE_Q6_K = 14 };
enum { ELEM_F32 = 0, ELEM_F16 = 1, ELEM_BF16 = 2 };
constexpr int ERR_UNSUPPORTED = -1;
constexpr int MATRIX_ROW_PADDING = 512;  // activation rows of the two-launch protocol are padded to this many values

// ---- the C ABI (include/inferencequant_b200.h) ----
using GemvFn = int (*)(int, int, const void*, const void*, void*, int, int, int, int, int, int, void*);
using GroupFn = int (*)(int, const int*, const void* const*, void* const*, const int*, int, int, const void*, int, void*);
using GemmWsFn = int (*)(int, int, const void*, const void*, void*, int, int, int, int, int, void*, int64_t, void*);
using MmqWsFn = int (*)(int, int, const void*, const void*, void*, int, int, int, int, void*, int64_t, void*);
using GemmBytesFn = int64_t (*)(int, int, int, int);
using GemvTcFn = int (*)(int, int, const void*, const void*, void*, int, int, int, int, int, void*, int64_t, void*);
using GemvTcBytesFn = int64_t (*)(int, int);
using QuantizeFn = int (*)(int, const void*, void*, int64_t, void*);
using DequantizeFn = int (*)(int, int, const void*, void*, int64_t, int, void*);
using GetRowsFn = int (*)(int, int, const void*, const int32_t*, void*, int64_t, int, int64_t, void*);
using StatusFn = int (*)();
using QuantQ8Fn = void (*)(const void*, void*, int, int, int, void*);
using PlainFn = void (*)(const void*, const void*, void*, int, int, int, int, int, void*);
using GluFn = void (*)(const void*, const void*, const void*, void*, int, int, int, int, int, int, void*);
using QuantMmqFn = void (*)(const void*, const int32_t*, void*, int, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, void*);
using MmqFn = void (*)(void*, const void*, const void*, void*, int64_t, int64_t, int64_t, int64_t, int64_t, int, int, int64_t, int, int, void*);

using Int8QuantizeFn = int (*)(int, const void*, int64_t, void*, int64_t, float*, int64_t, int, void*);
using Int8DequantizeFn = int (*)(int, const void*, int64_t, const float*, void*, int64_t, int, void*);
using Int8BytesFn = int64_t (*)(int, int);
using Int8MatmulFn = int (*)(int, const void*, const void*, const float*, void*, int, int, int, int64_t, int64_t, int64_t, void*, int64_t, void*);
using Int8ExpertsBytesFn = int64_t (*)(int, int, int, int, int, int);
using Int8ExpertsFn = int (*)(int, int, const void*, int64_t, const void*, int, const float*, const void*, const float*, const void*, const float*, void*, int, int, int,
                              int, int, void*, int64_t, void*);
using RouteSortFn = int (*)(const void*, int, int, int, int*, int*, int*, void*);
using RouteDispatchFn = int (*)(int, const void*, int64_t, const int*, const int*, int, void*, int, int, int, void*);
using RouteCombineFn = int (*)(int, int, const void*, int64_t, const int*, const float*, void*, int, int, int, void*);
using RouteCombineGradFn = int (*)(int, int, const void*, int64_t, const void*, int64_t, const int*, const int*, int, const float*, void*, float*, int, int, int, void*);
using LastErrorFn = const char* (*)();

// indexed by type (0 q8_0, 1 q4_k, 2 q6_k) and element type
struct Abi {
    GemvFn gemv;
    GroupFn group;
    GemmWsFn gemm_ws;
    GemmBytesFn gemm_bytes, mmq_bytes;
    MmqWsFn mmq_ws;
    GemvTcFn gemv_tc;
    GemvTcBytesFn gemv_tc_bytes;
    QuantizeFn quantize;
    DequantizeFn dequantize;
    GetRowsFn get_rows;
    StatusFn take_status;
    QuantQ8Fn quant_q8[3];
    PlainFn plain[3][3];
    GluFn glu[3][3];
    QuantMmqFn quant_mmq[2];  // D4, DS4
    MmqFn mmq[3];
    Int8QuantizeFn int8_quantize;
    Int8DequantizeFn int8_dequantize;
    Int8BytesFn int8_matmul_bytes;
    Int8MatmulFn int8_matmul;
    Int8ExpertsBytesFn int8_experts_bytes;
    Int8ExpertsFn int8_experts;
    RouteSortFn route_sort;
    RouteDispatchFn route_dispatch;
    RouteCombineFn route_combine;
    RouteCombineGradFn route_combine_grad;
    LastErrorFn last_error;
} abi{};
PyObject* check_fn = nullptr;          // kernel_library.check(rc, what): raises for a non-zero status
PyObject* launch_failed_fn = nullptr;  // raises for a status kept by a void launcher

struct AbiEntry {
    const char* name;
    void** slot;
};
const AbiEntry abi_entries[] = {
    {"b200q_gemv", (void**)&abi.gemv},
    {"b200q_gemv_group_act", (void**)&abi.group},
    {"b200q_gemm_ws", (void**)&abi.gemm_ws},
    {"b200q_mmq_ws", (void**)&abi.mmq_ws},
    {"b200q_mmq_workspace_bytes", (void**)&abi.mmq_bytes},
    {"b200q_gemm_workspace_bytes", (void**)&abi.gemm_bytes},
    {"b200q_gemv_tc", (void**)&abi.gemv_tc},
    {"b200q_gemv_tc_workspace_bytes", (void**)&abi.gemv_tc_bytes},
    {"b200q_quantize", (void**)&abi.quantize},
    {"b200q_dequantize", (void**)&abi.dequantize},
    {"b200q_get_rows", (void**)&abi.get_rows},
    {"b200q_take_launch_status", (void**)&abi.take_status},
    {"launch_mmvq_gguf_quantize_q8_1_f32", (void**)&abi.quant_q8[ELEM_F32]},
    {"launch_mmvq_gguf_quantize_q8_1_f16", (void**)&abi.quant_q8[ELEM_F16]},
    {"launch_mmvq_gguf_quantize_q8_1_bf16", (void**)&abi.quant_q8[ELEM_BF16]},
#define B200Q_HOST_TYPE(i, tag)                                              \
    {"launch_mmvq_gguf_" tag "_f32_plain", (void**)&abi.plain[i][ELEM_F32]},     \
    {"launch_mmvq_gguf_" tag "_f16_plain", (void**)&abi.plain[i][ELEM_F16]},     \
    {"launch_mmvq_gguf_" tag "_bf16_plain", (void**)&abi.plain[i][ELEM_BF16]},   \
    {"launch_mmvq_gguf_" tag "_f32_fused_glu", (void**)&abi.glu[i][ELEM_F32]},   \
    {"launch_mmvq_gguf_" tag "_f16_fused_glu", (void**)&abi.glu[i][ELEM_F16]},   \
    {"launch_mmvq_gguf_" tag "_bf16_fused_glu", (void**)&abi.glu[i][ELEM_BF16]}, \
    {"launch_mmq_gguf_" tag, (void**)&abi.mmq[i]},
    B200Q_HOST_TYPE(0, "q8_0") B200Q_HOST_TYPE(1, "q4_k") B200Q_HOST_TYPE(2, "q6_k")
#undef B200Q_HOST_TYPE
    {"launch_mmq_quantize_q8_1_D4", (void**)&abi.quant_mmq[0]},
    {"launch_mmq_quantize_q8_1_DS4", (void**)&abi.quant_mmq[1]},
    {"b200q_int8_quantize", (void**)&abi.int8_quantize},
    {"b200q_int8_dequantize", (void**)&abi.int8_dequantize},
    {"b200q_int8_matmul_workspace_bytes", (void**)&abi.int8_matmul_bytes},
    {"b200q_int8_matmul", (void**)&abi.int8_matmul},
    {"b200q_int8_experts_workspace_bytes", (void**)&abi.int8_experts_bytes},
    {"b200q_int8_experts", (void**)&abi.int8_experts},
    {"b200q_route_sort", (void**)&abi.route_sort},
    {"b200q_route_dispatch", (void**)&abi.route_dispatch},
    {"b200q_route_combine", (void**)&abi.route_combine},
    {"b200q_route_combine_grad", (void**)&abi.route_combine_grad},
    {"b200q_last_error", (void**)&abi.last_error},
};

int type_index(long type) { return type == TYPE_Q8_0 ? 0 : (type == TYPE_Q4_K ? 1 : (type == TYPE_Q6_K ? 2 : -1)); }
int64_t block_elems(int ti) { return ti == 0 ? 32 : 256; }
int64_t block_bytes(int ti) { return ti == 0 ? 34 : (ti == 1 ? 144 : 210); }
int elem_of(ScalarType t) {
    return t == ScalarType::Float ? ELEM_F32 : (t == ScalarType::Half ? ELEM_F16 : (t == ScalarType::BFloat16 ? ELEM_BF16 : -1));
}
int mmq_type_x(int elem) { return elem == ELEM_F32 ? 0 : (elem == ELEM_F16 ? 1 : 30); }
int64_t pad(int64_t k, int64_t to) { return (k + to - 1) / to * to; }

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

// ---- arguments ----
const Tensor* tensor_arg(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
bool cuda_contiguous(const Tensor* t) { return t != nullptr && t->is_cuda() && t->is_contiguous(); }
// anything that counts as an integer (a numpy integer has an index too)
bool int_arg(PyObject* o, long& v) {
    PyObject* i = PyNumber_Index(o);
    if (i != nullptr) {
        v = PyLong_AsLong(i);
        Py_DECREF(i);
    }
    if (i != nullptr && !(v == -1 && PyErr_Occurred())) return true;
    PyErr_Clear();
    return false;
}
bool int_args(PyObject* const* args, std::initializer_list<std::pair<int, long*>> list) {
    for (const auto& [i, v] : list)
        if (!int_arg(args[i], *v)) return false;
    return true;
}
Tensor empty(at::IntArrayRef size, ScalarType t, const Tensor& like) { return at::detail::empty_cuda(size, t, like.device(), std::nullopt); }
PyObject* none() { Py_RETURN_NONE; }
// a tuple that takes its items over
PyObject* tuple_of(std::initializer_list<PyObject*> items) {
    PyObject* tuple = PyTuple_New((Py_ssize_t)items.size());
    Py_ssize_t i = 0;
    for (PyObject* o : items) {
        if (tuple != nullptr) PyTuple_SET_ITEM(tuple, i++, o);
        else Py_XDECREF(o);
    }
    return tuple;
}
// launches may block (a full queue, a first load of a kernel): other Python threads go on meanwhile
struct NoGil {
    PyThreadState* state = PyEval_SaveThread();
    ~NoGil() { PyEval_RestoreThread(state); }
};
template <typename Fn, typename... Args> auto call(Fn fn, Args... args) {
    NoGil nogil;
    return fn(args...);
}

// 0: fine; otherwise a Python exception is set (kernel_library.check raises)
int failed(int rc, const char* what) {
    if (rc == 0) return 0;
    PyObject* r = PyObject_CallFunction(check_fn, "is", rc, what);
    Py_XDECREF(r);
    return 1;
}
int launcher_failed(const char* what) {
    const int rc = abi.take_status();
    if (rc == 0) return 0;
    PyObject* r = PyObject_CallFunction(launch_failed_fn, "is", rc, what);
    Py_XDECREF(r);
    return 1;
}

// ---- matmul ----
// quantize to Q8_1, then the reference's own matvec: shapes the one-launch kernel declines
int two_launches(int ti, int elem, const Tensor& w, const Tensor& x, Tensor& y, int64_t n, int64_t k, int64_t rows) {
    const int64_t kp = pad(k, MATRIX_ROW_PADDING);
    Tensor vy = empty({rows, kp / 32 * 36}, ScalarType::Byte, x);
    call(abi.quant_q8[elem], x.data_ptr(), vy.data_ptr(), (int)k, (int)kp, (int)rows, stream());
    call(abi.plain[ti][elem], w.data_ptr(), vy.data_ptr(), y.data_ptr(), (int)k, (int)n, (int)(kp / 32), (int)n, (int)rows, stream());
    return launcher_failed("launch_mmvq_gguf_*_plain");
}

// A workspace from the caching allocator for the duration of a call (given back in stream order); undefined if none is needed or the
// memory is not there, where the caller has a form that needs none.
Tensor workspace(int64_t bytes, const Tensor& like) {
    if (bytes <= 0) return Tensor();
    try {
        return empty({bytes}, ScalarType::Byte, like);
    } catch (const c10::OutOfMemoryError&) {
        return Tensor();
    }
}

// the tile GEMM
int gemm(long type, int elem, const Tensor& w, const Tensor& x, Tensor& y, int64_t m, int64_t n, int64_t k, int64_t ldx, int64_t ldy) {
    const int64_t bytes = abi.gemm_bytes((int)type, (int)m, (int)n, (int)k);
    const Tensor ws = workspace(bytes, x);
    return call(abi.gemm_ws, (int)type, elem, w.data_ptr(), x.data_ptr(), y.data_ptr(), (int)m, (int)n, (int)k, (int)ldx, (int)ldy,
                ws.defined() ? ws.data_ptr() : nullptr, bytes, stream());
}

// forward(type, w, n, k, x, act_quant, tier): y = x . W^T for contiguous x [..., k]; `tier` is what the caller's routing chose for
// the row count: 0 decode matvec, 1 small-batch tensor-core kernel, 2 tile GEMM, 3 as 1 or, where that refuses the weights or finds no room for its workspace, as 0
PyObject* py_forward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    long type, n, k, act_quant, tier;
    if (nargs != 7 || !int_args(args, {{0, &type}, {2, &n}, {3, &k}, {5, &act_quant}, {6, &tier}})) return none();
    const Tensor *w = tensor_arg(args[1]), *x = tensor_arg(args[4]);
    const int ti = type_index(type);
    if (ti < 0 || !cuda_contiguous(w) || !cuda_contiguous(x) || x->dim() < 2 || x->size(-1) != k || x->device() != w->device()) return none();
    const int elem = elem_of(x->scalar_type());
    if (elem < 0) return none();
    const int64_t rows = x->numel() / k;
    if (rows == 0) return none();
    c10::SmallVector<int64_t, 6> shape(x->sizes().begin(), x->sizes().end());
    shape.back() = n;
    if (tier == 2) {
        if (k % 64 != 0) return none();
        // the tensor-core path takes 16-bit activations; f32 inputs are narrowed and the result widened again
        const Tensor x16 = elem == ELEM_F32 ? at::_to_copy(*x, ScalarType::BFloat16) : *x;
        Tensor y = empty(shape, x16.scalar_type(), *x);
        if (failed(gemm(type, elem == ELEM_F32 ? ELEM_BF16 : elem, *w, x16, y, rows, n, k, k, n), "b200q_gemm"))
            return nullptr;
        return THPVariable_Wrap(elem == ELEM_F32 ? at::_to_copy(y, ScalarType::Float) : y);
    }
    Tensor y = empty(shape, x->scalar_type(), *x);
    if (tier == 1 || tier == 3) {
        const int64_t bytes = abi.gemv_tc_bytes((int)type, (int)k);
        if (bytes <= 0) return none();
        const Tensor ws = tier == 1 ? empty({bytes}, ScalarType::Byte, *x) : workspace(bytes, *x);
        const int rc = !ws.defined() ? ERR_UNSUPPORTED
                                     : call(abi.gemv_tc, (int)type, elem, w->data_ptr(), x->data_ptr(), y.data_ptr(), (int)rows, (int)n, (int)k, (int)k, (int)n,
                                            ws.data_ptr(), bytes, stream());
        if (rc != ERR_UNSUPPORTED || tier == 1) return failed(rc, "b200q_gemv_tc") ? nullptr : THPVariable_Wrap(std::move(y));
    }
    if (k % 128 == 0) {
        const int rc = call(abi.gemv, (int)type, elem, w->data_ptr(), x->data_ptr(), y.data_ptr(), (int)k, (int)n, (int)k, (int)n, (int)rows, (int)act_quant, stream());
        // no staged plan for this call (unaligned weights, no ring that fits): the two-launch protocol serves Q8_1 activations
        if (rc != ERR_UNSUPPORTED || act_quant != 0) return failed(rc, "b200q_gemv") ? nullptr : THPVariable_Wrap(std::move(y));
    } else if (act_quant != 0) {
        return none();
    }
    return two_launches(ti, elem, *w, *x, y, n, k, rows) ? nullptr : THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// gemv(type, w, x, n, out or None, act_quant)
PyObject* py_gemv(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    long type, n, act_quant;
    if (nargs != 6 || !int_args(args, {{0, &type}, {3, &n}, {5, &act_quant}})) return none();
    const Tensor *w = tensor_arg(args[1]), *x = tensor_arg(args[2]), *out = args[4] == Py_None ? nullptr : tensor_arg(args[4]);
    if (!cuda_contiguous(w) || !cuda_contiguous(x) || x->dim() != 2 || (args[4] != Py_None && (out == nullptr || out->dim() != 2))) return none();
    const int elem = elem_of(x->scalar_type());
    if (elem < 0) return none();
    const int64_t b = x->size(0), k = x->size(1);
    Tensor y = out != nullptr ? *out : empty({b, n}, x->scalar_type(), *x);
    if (failed(call(abi.gemv, (int)type, elem, w->data_ptr(), x->data_ptr(), y.data_ptr(), (int)k, (int)n, (int)x->stride(0), (int)y.stride(0), (int)b, (int)act_quant,
                        stream()),
               "b200q_gemv"))
        return nullptr;
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// gemm(type, w, x, n, out or None)
PyObject* py_gemm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    long type, n;
    if (nargs != 5 || !int_args(args, {{0, &type}, {3, &n}})) return none();
    const Tensor *w = tensor_arg(args[1]), *x = tensor_arg(args[2]), *out = args[4] == Py_None ? nullptr : tensor_arg(args[4]);
    if (!cuda_contiguous(w) || !cuda_contiguous(x) || x->dim() != 2 || (args[4] != Py_None && (out == nullptr || out->dim() != 2))) return none();
    const int elem = elem_of(x->scalar_type());
    if (elem < 0) return none();
    Tensor y = out != nullptr ? *out : empty({x->size(0), n}, x->scalar_type(), *x);
    if (failed(gemm(type, elem, *w, *x, y, x->size(0), n, x->size(1), x->stride(0), y.stride(0)), "b200q_gemm")) return nullptr;
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// gemv_group(types, ws, x, ns, outs or None, act_quant): lists of 1..4
PyObject* py_gemv_group(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    constexpr int MAX = 4;
    long act_quant;
    if (nargs != 6 || !int_arg(args[5], act_quant)) return none();
    for (int i : {0, 1, 3})
        if (!PyList_Check(args[i]) && !PyTuple_Check(args[i])) return none();
    const Tensor* x = tensor_arg(args[2]);
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(args[1]);
    const bool have_outs = args[4] != Py_None;
    if (n < 1 || n > MAX || PySequence_Fast_GET_SIZE(args[0]) != n || PySequence_Fast_GET_SIZE(args[3]) != n || !cuda_contiguous(x) || x->dim() != 2 ||
        x->size(0) != 1 || (have_outs && ((!PyList_Check(args[4]) && !PyTuple_Check(args[4])) || PySequence_Fast_GET_SIZE(args[4]) != n)))
        return none();
    const int elem = elem_of(x->scalar_type());
    if (elem < 0) return none();
    int types[MAX], ns[MAX];
    const void* ws[MAX];
    void* dsts[MAX];
    Tensor outs[MAX];
    for (Py_ssize_t i = 0; i < n; ++i) {
        long t, rows;
        if (!int_arg(PySequence_Fast_GET_ITEM(args[0], i), t) || !int_arg(PySequence_Fast_GET_ITEM(args[3], i), rows)) return none();
        const Tensor* w = tensor_arg(PySequence_Fast_GET_ITEM(args[1], i));
        if (!cuda_contiguous(w)) return none();
        types[i] = (int)t;
        ns[i] = (int)rows;
        ws[i] = w->data_ptr();
        if (have_outs) {
            const Tensor* o = tensor_arg(PySequence_Fast_GET_ITEM(args[4], i));
            if (o == nullptr) return none();
            dsts[i] = o->data_ptr();
        }
    }
    if (!have_outs)
        for (Py_ssize_t i = 0; i < n; ++i) {
            outs[i] = empty({1, (int64_t)ns[i]}, x->scalar_type(), *x);
            dsts[i] = outs[i].data_ptr();
        }
    const int rc = call(abi.group, (int)n, types, ws, dsts, ns, (int)x->size(1), elem, x->data_ptr(), (int)act_quant, stream());
    if (failed(rc, act_quant ? "b200q_gemv_group_act" : "b200q_gemv_group")) return nullptr;
    if (have_outs) {
        Py_INCREF(args[4]);
        return args[4];
    }
    PyObject* list = PyList_New(n);
    for (Py_ssize_t i = 0; list != nullptr && i < n; ++i) PyList_SET_ITEM(list, i, THPVariable_Wrap(std::move(outs[i])));
    return list;
    END_HANDLE_TH_ERRORS
}

// ---- the reference host's own sequence ----
// quantize_q8_1(x, k_padded)
PyObject* py_quantize_q8_1(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    long kp;
    if (nargs != 2 || !int_arg(args[1], kp)) return none();
    const Tensor* x = tensor_arg(args[0]);
    if (!cuda_contiguous(x) || x->dim() != 2 || elem_of(x->scalar_type()) < 0) return none();
    Tensor out = empty({x->size(0), kp / 32 * 36}, ScalarType::Byte, *x);
    call(abi.quant_q8[elem_of(x->scalar_type())], x->data_ptr(), out.data_ptr(), (int)x->size(1), (int)kp, (int)x->size(0), stream());
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// elem code of an output type given as its code
bool elem_scalar(long elem, ScalarType& t) {
    if (elem < 0 || elem > 2) return false;
    t = elem == ELEM_F32 ? ScalarType::Float : (elem == ELEM_F16 ? ScalarType::Half : ScalarType::BFloat16);
    return true;
}

// mmvq_plain(type, w, vy, n, k, b, elem, k_padded)
PyObject* py_mmvq_plain(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    long type, n, k, b, elem, kp;
    ScalarType t;
    if (nargs != 8 || !int_args(args, {{0, &type}, {3, &n}, {4, &k}, {5, &b}, {6, &elem}, {7, &kp}}) || !elem_scalar(elem, t)) return none();
    const Tensor *w = tensor_arg(args[1]), *vy = tensor_arg(args[2]);
    const int ti = type_index(type);
    if (ti < 0 || !cuda_contiguous(w) || !cuda_contiguous(vy)) return none();
    Tensor y = empty({b, n}, t, *w);
    call(abi.plain[ti][elem], w->data_ptr(), vy->data_ptr(), y.data_ptr(), (int)k, (int)n, (int)(kp / 32), (int)n, (int)b, stream());
    return launcher_failed("launch_mmvq_gguf_*_plain") ? nullptr : THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// mmvq_fused_glu(type, w_gate, w_up, vy, n, k, b, elem, k_padded, activation)
PyObject* py_mmvq_fused_glu(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    long type, n, k, b, elem, kp, act;
    ScalarType t;
    if (nargs != 10 || !int_args(args, {{0, &type}, {4, &n}, {5, &k}, {6, &b}, {7, &elem}, {8, &kp}, {9, &act}}) || !elem_scalar(elem, t)) return none();
    const Tensor *wg = tensor_arg(args[1]), *wu = tensor_arg(args[2]), *vy = tensor_arg(args[3]);
    const int ti = type_index(type);
    if (ti < 0 || !cuda_contiguous(wg) || !cuda_contiguous(wu) || !cuda_contiguous(vy)) return none();
    Tensor y = empty({b, n}, t, *vy);
    call(abi.glu[ti][elem], wg->data_ptr(), wu->data_ptr(), vy->data_ptr(), y.data_ptr(), (int)k, (int)n, (int)(kp / 32), (int)n, (int)b, (int)act, stream());
    return launcher_failed("launch_mmvq_gguf_*_fused_glu") ? nullptr : THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// quantize_mmq_q8_1(x, ds4, k_padded)
PyObject* py_quantize_mmq_q8_1(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    long ds4, kp;
    if (nargs != 3 || !int_args(args, {{1, &ds4}, {2, &kp}})) return none();
    const Tensor* x = tensor_arg(args[0]);
    if (!cuda_contiguous(x) || x->dim() != 2 || elem_of(x->scalar_type()) < 0) return none();
    const int64_t rows = x->size(0), k = x->size(1);
    Tensor out = empty({kp / 128, rows, 144}, ScalarType::Byte, *x);
    call(abi.quant_mmq[ds4 ? 1 : 0], x->data_ptr(), nullptr, out.data_ptr(), mmq_type_x(elem_of(x->scalar_type())), k, k, 0, 0, kp, rows, 1, 1, stream());
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// mmq(type, w, vy, m, n, k, elem, cc, nsm)
PyObject* py_mmq(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    long type, m, n, k, elem, cc, nsm;
    ScalarType t;
    if (nargs != 9 || !int_args(args, {{0, &type}, {3, &m}, {4, &n}, {5, &k}, {6, &elem}, {7, &cc}, {8, &nsm}}) || !elem_scalar(elem, t)) return none();
    const Tensor *w = tensor_arg(args[1]), *vy = tensor_arg(args[2]);
    const int ti = type_index(type);
    if (ti < 0 || !cuda_contiguous(w) || !cuda_contiguous(vy)) return none();
    Tensor y = empty({m, n}, t, *w);
    const int64_t bytes = abi.mmq_bytes((int)type, (int)m, (int)n, (int)k);
    if (const Tensor ws = workspace(bytes, *w); ws.defined()) {
        const int rc = call(abi.mmq_ws, (int)type, (int)elem, w->data_ptr(), vy->data_ptr(), y.data_ptr(), (int)m, (int)n, (int)k, (int)n, ws.data_ptr(), bytes,
                            stream());
        if (rc != ERR_UNSUPPORTED) return failed(rc, "b200q_mmq_ws") ? nullptr : THPVariable_Wrap(std::move(y));
    }
    call(abi.mmq[ti], nullptr, w->data_ptr(), vy->data_ptr(), y.data_ptr(), k, n, m, k / block_elems(ti), n, (int)cc, (int)nsm, 232448, 32, mmq_type_x((int)elem),
                stream());
    return launcher_failed("launch_mmq_gguf_*") ? nullptr : THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// ---- weights ----
// quantize(type, x): f32 [n, k] -> packed blocks, then the padding, zeroed
PyObject* py_quantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    long type;
    if (nargs != 2 || !int_arg(args[0], type)) return none();
    const Tensor* x = tensor_arg(args[1]);
    const int ti = type_index(type);
    if (ti < 0 || !cuda_contiguous(x) || x->dim() != 2 || x->scalar_type() != ScalarType::Float || x->size(1) % block_elems(ti) != 0) return none();
    const int64_t bytes = x->numel() / block_elems(ti) * block_bytes(ti), padding = MATRIX_ROW_PADDING / block_elems(ti) * block_bytes(ti);
    Tensor buf = empty({bytes + padding}, ScalarType::Byte, *x);
    buf.narrow(0, bytes, padding).zero_();
    if (failed(call(abi.quantize, (int)type, x->data_ptr(), buf.data_ptr(), x->numel(), stream()), "b200q_quantize")) return nullptr;
    return THPVariable_Wrap(std::move(buf));
    END_HANDLE_TH_ERRORS
}

// dequantize(type, w, n, k, elem)
PyObject* py_dequantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    long type, n, k, elem;
    ScalarType t;
    if (nargs != 5 || !int_args(args, {{0, &type}, {2, &n}, {3, &k}, {4, &elem}}) || !elem_scalar(elem, t)) return none();
    const Tensor* w = tensor_arg(args[1]);
    if (!cuda_contiguous(w)) return none();
    Tensor out = empty({n, k}, t, *w);
    if (failed(call(abi.dequantize, (int)type, (int)elem, w->data_ptr(), out.data_ptr(), n, (int)k, stream()), "b200q_dequantize")) return nullptr;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// get_rows(type, w, ids, n, k, elem): ids int32, contiguous, on the device
PyObject* py_get_rows(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    long type, n, k, elem;
    ScalarType t;
    if (nargs != 6 || !int_args(args, {{0, &type}, {3, &n}, {4, &k}, {5, &elem}}) || !elem_scalar(elem, t)) return none();
    const Tensor *w = tensor_arg(args[1]), *ids = tensor_arg(args[2]);
    if (!cuda_contiguous(w) || !cuda_contiguous(ids) || ids->scalar_type() != ScalarType::Int || ids->device() != w->device()) return none();
    c10::SmallVector<int64_t, 6> shape(ids->sizes().begin(), ids->sizes().end());
    shape.push_back(k);
    Tensor out = empty(shape, t, *w);
    if (failed(call(abi.get_rows, (int)type, (int)elem, w->data_ptr(), static_cast<const int32_t*>(ids->data_ptr()), out.data_ptr(), ids->numel(), (int)k, n, stream()),
               "b200q_get_rows"))
        return nullptr;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ---- int8 rows, experts, routing ----
// These launch on the current stream of their tensors' device.
constexpr int64_t INT8_ROW_ALIGN = 16, MOST = 2147483647 - 65536;

struct OnDevice {
    c10::cuda::CUDAGuard guard;
    void* stream;
    explicit OnDevice(const Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};
bool same_device(const Tensor& a, std::initializer_list<const Tensor*> others) {
    for (const Tensor* t : others)
        if (t->device() != a.device()) return false;
    return true;
}
bool of(const Tensor* t, ScalarType type) { return cuda_contiguous(t) && t->scalar_type() == type; }
// rows of unit stride that do not overlap
bool row_stride(const Tensor& t, int64_t& ld) {
    if (t.dim() != 2) return false;
    if (t.is_contiguous()) {
        ld = t.size(1);
        return true;
    }
    ld = t.stride(0);
    return t.size(0) > 1 && t.size(1) > 1 && t.stride(1) == 1 && ld >= t.size(1);
}
bool wants_grad(const Tensor& t) { return t.requires_grad() && c10::GradMode::is_enabled(); }
// a derivative of forward mode, which is there without requires_grad and under no_grad too
bool has_tangent(const Tensor& t) { return t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode(); }
// in a backward pass there is no interpreter to raise with
void require(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed with status ", rc, ": ", abi.last_error()); }

// int8_forward(wq, scales, n, k, x): y = x . W^T
PyObject* py_int8_forward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    long n, k;
    if (nargs != 5 || !int_args(args, {{2, &n}, {3, &k}})) return none();
    const Tensor *w = tensor_arg(args[0]), *ws = tensor_arg(args[1]), *x = tensor_arg(args[4]);
    if (!of(w, ScalarType::Char) || !of(ws, ScalarType::Float) || !cuda_contiguous(x) || x->dim() < 2 || x->size(-1) != k || k < 1 || k > MOST || n < 1 || n > MOST || wants_grad(*x) || has_tangent(*x)) return none();
    const int64_t kp = pad(k, INT8_ROW_ALIGN), m = x->numel() / k;
    const int elem = elem_of(x->scalar_type());
    if (elem < 0 || m == 0 || m > MOST || w->dim() != 2 || w->size(0) != n || w->size(1) != kp || ws->numel() != n || !same_device(*x, {w, ws})) return none();
    OnDevice on(*x);
    c10::SmallVector<int64_t, 6> shape(x->sizes().begin(), x->sizes().end());
    shape.back() = n;
    Tensor y = empty(shape, x->scalar_type(), *x);
    const int64_t bytes = abi.int8_matmul_bytes((int)m, (int)k);
    const Tensor space = empty({bytes}, ScalarType::Byte, *x);
    if (failed(call(abi.int8_matmul, elem, x->data_ptr(), w->data_ptr(), ws->data_ptr<float>(), y.data_ptr(), (int)m, (int)n, (int)k, (int64_t)k, kp, (int64_t)n, space.data_ptr(), bytes,
                    on.stream),
               "b200q_int8_matmul"))
        return nullptr;
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// int8_quantize(x): (q, scales) of a matrix's rows
PyObject* py_int8_quantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    const Tensor* x = nargs == 1 ? tensor_arg(args[0]) : nullptr;
    int64_t ld;
    if (x == nullptr || !x->is_cuda() || !row_stride(*x, ld) || elem_of(x->scalar_type()) < 0 || x->numel() == 0 || x->size(0) > MOST || x->size(1) > MOST) return none();
    OnDevice on(*x);
    const int64_t m = x->size(0), k = x->size(1), kp = pad(k, INT8_ROW_ALIGN);
    Tensor q = empty({m, kp}, ScalarType::Char, *x), scales = empty({m}, ScalarType::Float, *x);
    if (failed(call(abi.int8_quantize, elem_of(x->scalar_type()), x->data_ptr(), ld, q.data_ptr(), kp, scales.data_ptr<float>(), m, (int)k, on.stream), "b200q_int8_quantize"))
        return nullptr;
    return tuple_of({THPVariable_Wrap(std::move(q)), THPVariable_Wrap(std::move(scales))});
    END_HANDLE_TH_ERRORS
}

// int8_dequantize(q, scales, k, elem)
PyObject* py_int8_dequantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    long k, elem;
    ScalarType t;
    if (nargs != 4 || !int_args(args, {{2, &k}, {3, &elem}}) || !elem_scalar(elem, t)) return none();
    const Tensor *q = tensor_arg(args[0]), *scales = tensor_arg(args[1]);
    if (!of(q, ScalarType::Char) || !of(scales, ScalarType::Float) || q->dim() < 2 || k < 1 || k > MOST || q->size(-1) != pad(k, INT8_ROW_ALIGN) || q->numel() == 0 || !same_device(*q, {scales})) return none();
    const int64_t rows = q->numel() / q->size(-1);
    if (scales->numel() != rows || rows > MOST) return none();
    OnDevice on(*q);
    c10::SmallVector<int64_t, 6> shape(q->sizes().begin(), q->sizes().end());
    shape.back() = k;
    Tensor out = empty(shape, t, *q);
    if (failed(call(abi.int8_dequantize, (int)elem, q->data_ptr(), q->size(-1), scales->data_ptr<float>(), out.data_ptr(), rows, (int)k, on.stream), "b200q_int8_dequantize")) return nullptr;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// int8_experts(x, ids, weights, gate_up, gate_up_scales, down, down_scales, ffn, activation)
PyObject* py_int8_experts(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    long ffn, act;
    if (nargs != 9 || !int_args(args, {{7, &ffn}, {8, &act}})) return none();
    const Tensor* t[7];
    for (int i = 0; i < 7; ++i)
        if (!cuda_contiguous(t[i] = tensor_arg(args[i]))) return none();
    const Tensor &x = *t[0], &ids = *t[1], &weights = *t[2], &gate_up = *t[3], &gus = *t[4], &down = *t[5], &ds = *t[6];
    const int elem = elem_of(x.scalar_type());
    if (elem < 0 || (ids.scalar_type() != ScalarType::Int && ids.scalar_type() != ScalarType::Long) || weights.scalar_type() != ScalarType::Float ||
        gate_up.scalar_type() != ScalarType::Char || down.scalar_type() != ScalarType::Char || gus.scalar_type() != ScalarType::Float || ds.scalar_type() != ScalarType::Float ||
        x.dim() < 2 || ids.dim() != x.dim() || ids.sizes() != weights.sizes() || gate_up.dim() != 3 || down.dim() != 3 || ffn < 1 || x.numel() == 0 || ids.numel() == 0 ||
        wants_grad(x) || wants_grad(weights) || has_tangent(x) || has_tangent(weights) || !same_device(x, {t[1], t[2], t[3], t[4], t[5], t[6]}))
        return none();
    for (int64_t i = 0; i + 1 < x.dim(); ++i)
        if (x.size(i) != ids.size(i)) return none();
    const int64_t hidden = x.size(-1), tokens = x.numel() / hidden, topk = ids.size(-1), experts = gate_up.size(0), p = pad(ffn, 8);
    if (tokens * topk > MOST || hidden > MOST || ffn > MOST || experts > MOST || gate_up.size(1) != 2 * p || gate_up.size(2) != pad(hidden, INT8_ROW_ALIGN) || down.size(0) != experts || down.size(1) != hidden ||
        down.size(2) != pad(ffn, INT8_ROW_ALIGN) || gus.numel() != experts * 2 * p || ds.numel() != experts * hidden)
        return none();
    OnDevice on(x);
    Tensor out = empty(x.sizes(), x.scalar_type(), x);
    const int64_t bytes = abi.int8_experts_bytes(elem, (int)tokens, (int)topk, (int)experts, (int)hidden, (int)ffn);
    const Tensor space = empty({bytes}, ScalarType::Byte, x);
    if (failed(call(abi.int8_experts, elem, (int)act, x.data_ptr(), hidden, ids.data_ptr(), (int)ids.element_size(), weights.data_ptr<float>(), gate_up.data_ptr(), gus.data_ptr<float>(),
                    down.data_ptr(), ds.data_ptr<float>(), out.data_ptr(), (int)tokens, (int)experts, (int)topk, (int)hidden, (int)ffn, space.data_ptr(), bytes, on.stream),
               "b200q_int8_experts"))
        return nullptr;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// route_sort(ids, experts): (order, offsets, position)
PyObject* py_route_sort(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    long experts;
    if (nargs != 2 || !int_arg(args[1], experts) || experts < 1 || experts > 1024) return none();
    const Tensor* ids = tensor_arg(args[0]);
    if (!cuda_contiguous(ids) || (ids->scalar_type() != ScalarType::Int && ids->scalar_type() != ScalarType::Long) || ids->numel() > MOST) return none();
    OnDevice on(*ids);
    const int64_t slots = ids->numel();
    Tensor order = empty({slots}, ScalarType::Int, *ids), offsets = empty({experts + 1}, ScalarType::Int, *ids), position = empty(ids->sizes(), ScalarType::Int, *ids);
    if (failed(call(abi.route_sort, ids->data_ptr(), (int)ids->element_size(), (int)slots, (int)experts, order.data_ptr<int>(), offsets.data_ptr<int>(), position.data_ptr<int>(), on.stream),
               "b200q_route_sort"))
        return nullptr;
    return tuple_of({THPVariable_Wrap(std::move(order)), THPVariable_Wrap(std::move(offsets)), THPVariable_Wrap(std::move(position))});
    END_HANDLE_TH_ERRORS
}

Tensor combine(const Tensor& rows, int64_t ld, const Tensor& position, const float* weights, ScalarType type) {
    const int64_t topk = position.size(-1), tokens = position.numel() / topk;
    OnDevice on(rows);
    Tensor out = empty({tokens, rows.size(1)}, type, rows);
    require(abi.route_combine(elem_of(rows.scalar_type()), elem_of(type), rows.data_ptr(), ld, position.data_ptr<int>(), weights, out.data_ptr(), (int)tokens, (int)topk, (int)rows.size(1),
                              on.stream),
            "b200q_route_combine");
    return out;
}
Tensor dispatch(const Tensor& x, int64_t ld, const Tensor& position, const Tensor& offsets) {
    const int64_t topk = position.size(-1);
    OnDevice on(x);
    Tensor rows = empty({x.size(0) * topk, x.size(1)}, x.scalar_type(), x);
    require(abi.route_dispatch(elem_of(x.scalar_type()), x.data_ptr(), ld, position.data_ptr<int>(), offsets.data_ptr<int>(), (int)offsets.numel() - 1, rows.data_ptr(), (int)x.size(0),
                               (int)topk, (int)x.size(1), on.stream),
            "b200q_route_dispatch");
    return rows;
}
// a gradient as the kernels take it
Tensor grad_rows_of(const Tensor& g, int64_t& ld) {
    if (row_stride(g, ld)) return g;
    Tensor c = g.contiguous();
    ld = c.size(1);
    return c;
}
void no_tangent(const Tensor& grad) { TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(grad), "the routing of tokens has no derivatives in forward mode, nor do its gradients"); }
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
// passes a gradient on that is not to be differentiated again
struct OnceFunction : torch::autograd::Function<OnceFunction> {
    static Tensor forward(AutogradContext*, const Tensor& grad) { return grad; }
    static variable_list backward(AutogradContext*, variable_list) { TORCH_CHECK(false, "the gradients of token routing cannot be differentiated again"); }
};
// A gradient made of `sources`: under create_graph one that raises if it is differentiated, towards whichever of them.
Tensor once(Tensor grad, std::initializer_list<const Tensor*> sources) {
    if (!grad.defined() || !c10::GradMode::is_enabled()) return grad;
    for (const Tensor* t : sources)
        if (t->requires_grad()) {
            grad.set_requires_grad(true);
            return OnceFunction::apply(grad);
        }
    return grad;
}
struct DispatchFunction : torch::autograd::Function<DispatchFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& position, const Tensor& offsets) {
        ctx->save_for_backward({position});
        ctx->saved_data["type"] = (int64_t)x.scalar_type();
        int64_t ld;
        TORCH_CHECK(row_stride(x, ld));  // the caller has looked
        return dispatch(x, ld, position, offsets);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor position = ctx->get_saved_variables()[0];
        no_tangent(grads[0]);
        int64_t ld;
        const Tensor g = grad_rows_of(grads[0], ld);
        return {once(combine(g, ld, position, nullptr, (ScalarType)ctx->saved_data["type"].toInt()), {&grads[0]}), Tensor(), Tensor()};
    }
};
struct CombineFunction : torch::autograd::Function<CombineFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& weights, const Tensor& position, const Tensor& offsets, int64_t type) {
        ctx->save_for_backward({rows, weights, position, offsets});
        int64_t ld;
        TORCH_CHECK(row_stride(rows, ld));
        return combine(rows, ld, position, weights.data_ptr<float>(), (ScalarType)type);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &rows = saved[0], &weights = saved[1], &position = saved[2], &offsets = saved[3];
        no_tangent(grads[0]);
        int64_t ldg, ldr;
        const Tensor g = grad_rows_of(grads[0], ldg);
        TORCH_CHECK(row_stride(rows, ldr));
        const int64_t topk = position.size(-1), tokens = position.numel() / topk;
        OnDevice on(g);
        Tensor grad_rows, grad_weights;
        if (ctx->needs_input_grad(0)) grad_rows = empty({rows.size(0), rows.size(1)}, rows.scalar_type(), rows);
        if (ctx->needs_input_grad(1)) grad_weights = empty(weights.sizes(), ScalarType::Float, rows);
        require(abi.route_combine_grad(elem_of(g.scalar_type()), elem_of(rows.scalar_type()), g.data_ptr(), ldg, rows.data_ptr(), ldr, position.data_ptr<int>(), offsets.data_ptr<int>(),
                                       (int)offsets.numel() - 1, weights.data_ptr<float>(), grad_rows.defined() ? grad_rows.data_ptr() : nullptr,
                                       grad_weights.defined() ? grad_weights.data_ptr<float>() : nullptr, (int)tokens, (int)topk, (int)rows.size(1), on.stream),
                "b200q_route_combine_grad");
        return {once(grad_rows, {&grads[0], &weights}), once(grad_weights, {&grads[0], &rows}), Tensor(), Tensor(), Tensor()};
    }
};

// route_dispatch(x, position, offsets), differentiable
PyObject* py_route_dispatch(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 3) return none();
    const Tensor *x = tensor_arg(args[0]), *position = tensor_arg(args[1]), *offsets = tensor_arg(args[2]);
    int64_t ld;
    if (x == nullptr || !x->is_cuda() || !row_stride(*x, ld) || elem_of(x->scalar_type()) < 0 || x->numel() == 0 || x->size(1) > MOST || !of(position, ScalarType::Int) || position->dim() < 2 ||
        position->numel() == 0 || position->numel() / position->size(-1) != x->size(0) || !of(offsets, ScalarType::Int) || offsets->numel() < 2 || !same_device(*x, {position, offsets}) || has_tangent(*x))
        return none();
    Tensor rows;
    {
        NoGil nogil;
        rows = wants_grad(*x) ? DispatchFunction::apply(*x, *position, *offsets) : dispatch(*x, ld, *position, *offsets);
    }
    return THPVariable_Wrap(std::move(rows));
    END_HANDLE_TH_ERRORS
}

// route_combine(rows, weights, position, offsets, elem), differentiable
PyObject* py_route_combine(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    long elem;
    ScalarType type;
    if (nargs != 5 || !int_arg(args[4], elem) || !elem_scalar(elem, type)) return none();
    const Tensor *rows = tensor_arg(args[0]), *weights = tensor_arg(args[1]), *position = tensor_arg(args[2]), *offsets = tensor_arg(args[3]);
    int64_t ld;
    if (rows == nullptr || !rows->is_cuda() || !row_stride(*rows, ld) || elem_of(rows->scalar_type()) < 0 || rows->numel() == 0 || rows->size(1) > MOST || !of(weights, ScalarType::Float) ||
        !of(position, ScalarType::Int) || position->dim() < 2 || position->sizes() != weights->sizes() || position->numel() != rows->size(0) || !of(offsets, ScalarType::Int) ||
        offsets->numel() < 2 || !same_device(*rows, {weights, position, offsets}) || has_tangent(*rows) || has_tangent(*weights))
        return none();
    Tensor out;
    {
        NoGil nogil;
        out = wants_grad(*rows) || wants_grad(*weights) ? CombineFunction::apply(*rows, *weights, *position, *offsets, (int64_t)type)
                                                        : combine(*rows, ld, *position, weights->data_ptr<float>(), type);
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// bind(names, addresses, check, launch_failed)
PyObject* py_bind(PyObject*, PyObject* args) {
    PyObject *addresses, *check, *launch_failed;
    if (!PyArg_ParseTuple(args, "O!OO", &PyDict_Type, &addresses, &check, &launch_failed)) return nullptr;
    for (const AbiEntry& e : abi_entries) {
        PyObject* v = PyDict_GetItemString(addresses, e.name);
        if (v == nullptr) return PyErr_Format(PyExc_KeyError, "no address for %s", e.name);
        *e.slot = PyLong_AsVoidPtr(v);
        if (PyErr_Occurred()) return nullptr;
    }
    Py_INCREF(check);
    Py_INCREF(launch_failed);
    Py_XSETREF(check_fn, check);
    Py_XSETREF(launch_failed_fn, launch_failed);
    Py_RETURN_NONE;
}

PyObject* py_symbols(PyObject*, PyObject*) {
    PyObject* list = PyList_New(0);
    for (const AbiEntry& e : abi_entries) {
        PyObject* s = PyUnicode_FromString(e.name);
        if (list == nullptr || s == nullptr || PyList_Append(list, s) != 0) return nullptr;
        Py_DECREF(s);
    }
    return list;
}

#define B200Q_FAST(name, fn) {name, (PyCFunction)(void (*)(void))fn, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    {"bind", py_bind, METH_VARARGS, nullptr},
    {"symbols", py_symbols, METH_NOARGS, nullptr},
    B200Q_FAST("forward", py_forward),
    B200Q_FAST("gemv", py_gemv),
    B200Q_FAST("gemv_group", py_gemv_group),
    B200Q_FAST("gemm", py_gemm),
    B200Q_FAST("quantize_q8_1", py_quantize_q8_1),
    B200Q_FAST("mmvq_plain", py_mmvq_plain),
    B200Q_FAST("mmvq_fused_glu", py_mmvq_fused_glu),
    B200Q_FAST("quantize_mmq_q8_1", py_quantize_mmq_q8_1),
    B200Q_FAST("mmq", py_mmq),
    B200Q_FAST("quantize", py_quantize),
    B200Q_FAST("dequantize", py_dequantize),
    B200Q_FAST("get_rows", py_get_rows),
    B200Q_FAST("int8_forward", py_int8_forward),
    B200Q_FAST("int8_quantize", py_int8_quantize),
    B200Q_FAST("int8_dequantize", py_int8_dequantize),
    B200Q_FAST("int8_experts", py_int8_experts),
    B200Q_FAST("route_sort", py_route_sort),
    B200Q_FAST("route_dispatch", py_route_dispatch),
    B200Q_FAST("route_combine", py_route_combine),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "b200q_torch_host", "Native call path of the torch front end.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_b200q_torch_host(void) { return PyModule_Create(&module_def); }
