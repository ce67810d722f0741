// lm_torch.h -- what the torch bindings of the language-model operators share: checks
// of arguments, tensors as rows, streams, and the ends of autograd nodes.
//
// Internal to _lm_torch.so; host code only.
#pragma once

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <algorithm>
#include <optional>
#include <utility>

#include "../../../include/spiky_lm.h"
#include "../../../include/spiky_lm_tokens.h"
#include "../../../include/spiky_lut.h"

namespace lm_torch {

using at::ScalarType;
using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// ---- checks and views -------------------------------------------------------
inline void check(int status) {
    if (status == SPIKY_OK) return;
    TORCH_CHECK_VALUE(status != SPIKY_VALUE_ERROR, spiky_lm_last_error());
    TORCH_CHECK(false, spiky_lm_last_error());
}

inline int type_code(ScalarType t) {
    return t == at::kFloat ? SPIKY_F32 : t == at::kBFloat16 ? SPIKY_BF16 : t == at::kHalf ? SPIKY_F16 : -1;
}

inline int type_code(const Tensor &t, const char *name) {
    const int code = type_code(t.scalar_type());
    TORCH_CHECK(code >= 0, "tensor ", name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
    return code;
}

// With its memory's values: torch keeps the sign of imaginary parts of conjugates beside them.
inline Tensor settled(const Tensor &t) { return t.is_neg() ? t.resolve_neg() : t; }

inline Tensor device_tensor(PyObject *o, const char *name) {
    TORCH_CHECK(THPVariable_Check(o), "tensor ", name, " must be a torch.Tensor");
    const Tensor &t = THPVariable_Unpack(o);
    TORCH_CHECK(t.device().is_cuda(), "tensor ", name, " must be on CUDA");
    return settled(t);
}

// A trace sees torch's own calls alone, and would keep the results here as constants.
inline void check_trace() {
    TORCH_CHECK(!at::tracer::impl::is_dispatch_enabled(),
                "spiky_amd's language-model operators cannot be traced by torch.jit.trace");
}

// Forward-mode derivatives are not computed, and a result without a tangent would count as constant.
inline void check_tangent(PyObject *o, const char *name) {
    TORCH_CHECK_NOT_IMPLEMENTED(!THPVariable_Check(o) || !THPVariable_Unpack(o)._fw_grad(0).defined(),
                                "spiky_amd's language-model operators have no forward-mode derivatives, but tensor ",
                                name, " has a tangent");
}

// Undefined for None.
inline Tensor device_tensor(PyObject *o, const char *name, c10::Device device) {
    if (o == Py_None) return Tensor();
    Tensor t = device_tensor(o, name);
    TORCH_CHECK(t.device() == device, "tensor ", name, " must be on ", device, ", got ", t.device());
    return t;
}

inline void *pointer(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

inline double number(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}

inline uint64_t bits64(PyObject *o) {
    THPObjectPtr index(PyNumber_Index(o));
    if (!index) throw python_error();
    const uint64_t v = PyLong_AsUnsignedLongLongMask(index.get());
    if (v == (uint64_t)-1 && PyErr_Occurred()) throw python_error();
    return v;
}

// A whole number of 64 bits with its sign.
inline int64_t whole(PyObject *o, const char *name) {
    THPObjectPtr index(PyNumber_Index(o));
    if (!index) throw python_error();
    int past = 0;
    const int64_t v = PyLong_AsLongLongAndOverflow(index.get(), &past);
    TORCH_CHECK_VALUE(!past, name, " must fit 64 bits");
    return v;
}

inline double probability(PyObject *o) {
    const double p = number(o);
    TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "dropout probability must be between 0 and 1, got ", p);
    return p;
}

struct Generator {
    uint64_t seed = 0, offset = 0;
    Tensor state;  // [seed, offset] in device memory, in their place
};

inline Generator generator(PyObject *seed, PyObject *offset, c10::Device device) {
    Generator g;
    if (!THPVariable_Check(seed)) {
        g.seed = bits64(seed);
        g.offset = bits64(offset);
        return g;
    }
    g.state = device_tensor(seed, "seed", device);
    TORCH_CHECK(g.state.scalar_type() == at::kLong && g.state.numel() == 2 && g.state.is_contiguous(),
                "tensor seed must be a contiguous int64 tensor of [seed, offset]");
    TORCH_CHECK_VALUE(bits64(offset) == 0, "offset is the second element of a seed tensor");
    return g;
}

// The tensor seen as rows of its last dimension, and the elements from row to
// row.  Rows at one distance with contiguous columns stay where they are; others
// are copied.
inline std::pair<Tensor, int64_t> as_rows(const Tensor &given) {
    const Tensor t = settled(given);
    const int64_t dim = t.dim();
    const int64_t cols = dim ? t.size(-1) : 1;
    if (t.is_contiguous()) return {t, cols};
    if (dim && t.stride(-1) == 1 && t.numel()) {
        int64_t step = -1, reach = 0;  // from the innermost dimension of more than one
        bool even = true;
        for (int64_t k = dim - 2; k >= 0; k--) {
            if (t.size(k) == 1) continue;
            if (step < 0)
                step = t.stride(k);
            else if (t.stride(k) != reach)
                even = false;
            reach = t.stride(k) * t.size(k);
        }
        if (even) return {t, step < 0 ? cols : step};
    }
    return {t.contiguous(), cols};
}

inline int64_t rows_of(const Tensor &t) {
    const int64_t cols = t.dim() ? t.size(-1) : 1;
    return cols ? t.numel() / cols : 0;
}

// An uninitialised tensor, without the dispatcher's way to the same call.
inline Tensor fresh(at::IntArrayRef sizes, ScalarType type, c10::Device device) {
    return at::detail::empty_cuda(sizes, type, device, std::nullopt);
}

struct OnDevice {
    c10::DeviceGuard guard;
    void *stream;
    explicit OnDevice(c10::Device d) : guard(d), stream(c10::hip::getCurrentHIPStream(d.index()).stream()) {}
};

// Gradients in a capture cannot go to a node that was recorded on the default stream
// (a leaf's, kept alive by an eager graph): autograd would make that stream wait for
// the captured one, which ends the process.  So the backward call raises first.
inline void check_capture(const Node &node, c10::Device device) {
    const c10::Stream standard = c10::hip::getDefaultHIPStream(device.index()).unwrap();
    if (c10::hip::getCurrentHIPStream(device.index()).unwrap() == standard) return;  // which is never captured
    bool stands = false;
    for (size_t i = 0; i < node.num_outputs(); i++) {
        if (!node.task_should_compute_output(i)) continue;
        const auto stream = node.next_edge(i).function->stream();
        stands = stands || (stream && stream->id() == standard.id() && stream->device_index() == device.index());
    }
    if (!stands) return;
    TORCH_CHECK(c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None,
                "a gradient belongs to the default stream, which a captured backward pass cannot reach: drop eager "
                "graphs of the same leaves before the capture, or run them on a side stream");
}

inline bool needs_grad(const Tensor &t) { return t.defined() && t.requires_grad(); }

// Gradients of the gradients are not computed: a backward pass through these raises.
struct Twice : Node {
    variable_list apply(variable_list &&) override {
        TORCH_CHECK(false, "spiky_amd's language-model operators cannot be differentiated twice");
    }
};

inline variable_list once_differentiable(variable_list &&grads, torch::autograd::edge_list &&inputs) {
    auto stop = std::make_shared<Twice>();
    stop->set_next_edges(std::move(inputs));  // so that a search for them comes by here
    for (Tensor &t : grads)
        if (t.defined()) torch::autograd::set_history(t, stop);
    return std::move(grads);
}

// Runs a node's gradients, and marks them where a graph of them is asked for: as of the node's inputs
// and of the outputs' gradients.
template <typename N>
struct Once : N {
    variable_list apply(variable_list &&grads) override {
        if (!at::GradMode::is_enabled()) return N::apply(std::move(grads));
        torch::autograd::edge_list inputs = N::next_edges();
        for (const Tensor &t : grads)
            if (t.defined() && t.requires_grad()) inputs.push_back(torch::autograd::impl::gradient_edge(t));
        return once_differentiable(N::apply(std::move(grads)), std::move(inputs));
    }
};

inline PyObject *pair(PyObject *first, PyObject *second) {
    PyObject *t = PyTuple_New(2);
    if (!t) throw python_error();
    PyTuple_SET_ITEM(t, 0, first);
    PyTuple_SET_ITEM(t, 1, second);
    return t;
}

inline PyObject *wrapped(const Tensor &t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_INCREF(Py_None);
    return Py_None;
}

// n rows of `width` bytes in memory, `step` bytes apart.
struct Span {
    uintptr_t at = 0;
    int64_t n = 0, step = 0, width = 0;
};

// The rows of a tensor with contiguous columns, `stride` elements apart; one row for all where that is 0.
inline Span span_of(const Tensor &t, int64_t stride) {
    if (!t.defined() || t.numel() == 0) return {};
    const int64_t size = (int64_t)t.element_size(), rows = t.dim() == 2 ? t.size(0) : 1;
    return {reinterpret_cast<uintptr_t>(t.data_ptr()), stride ? rows : 1, stride * size, t.size(-1) * size};
}

// Rows of both are in the order of their addresses, so one walk along them meets any two that overlap.
inline bool overlap(const Span &a, const Span &b) {
    if (a.at + (a.n - 1) * a.step + a.width <= b.at || b.at + (b.n - 1) * b.step + b.width <= a.at) return false;
    for (int64_t i = 0, j = 0; i < a.n && j < b.n;) {
        const uintptr_t from_a = a.at + i * a.step, from_b = b.at + j * b.step;
        if (from_a + a.width <= from_b)
            i++;
        else if (from_b + b.width <= from_a)
            j++;
        else
            return true;
    }
    return false;
}

inline bool is_index(const Tensor &t, const char *name) {
    const bool wide = t.scalar_type() == at::kLong;
    TORCH_CHECK(wide || t.scalar_type() == at::kInt, "tensor ", name, " must have dtype int32 or int64, got ",
                t.scalar_type());
    return wide;
}

// [n] for every row, or [rows, n]: with contiguous columns, and the distance of its rows.
inline std::pair<Tensor, int64_t> by_row(const Tensor &t, const char *name, int64_t rows) {
    TORCH_CHECK_VALUE(t.dim() == 1 || (t.dim() == 2 && t.size(0) == rows), name, " must be [n] or [", rows,
                      ", n], got ", t.sizes());
    if (t.dim() == 1) return {t.contiguous(), 0};
    Tensor c = t.size(1) > 1 && t.stride(1) != 1 ? t.contiguous() : t;
    const int64_t stride = c.stride(0);
    return {c, stride};
}

// ---- the operators of lm_tokens_torch.cpp ------------------------------------
PyObject *embed_tokens(PyObject *, PyObject *const *args, Py_ssize_t n);
PyObject *beam_select(PyObject *, PyObject *const *args, Py_ssize_t n);
PyObject *reorder_states(PyObject *, PyObject *const *args, Py_ssize_t n);

}  // namespace lm_torch
