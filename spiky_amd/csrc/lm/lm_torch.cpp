// lm_torch.cpp -- the operators of include/spiky_lm.h on torch tensors: checks of
// arguments, outputs, streams and autograd.  Host code only; all device work goes
// through the C ABI of libspiky_lut.so.
//
// A training step of a small model is bound by what the host does between
// launches.  Python functions over ctypes took 92-103 us for a pass of the
// residual join and its gradients whose kernels take 33.
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
#include "../../../include/spiky_lut.h"

namespace {

using at::ScalarType;
using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// ---- checks and views -------------------------------------------------------
void check(int status) {
    if (status == SPIKY_OK) return;
    TORCH_CHECK_VALUE(status != SPIKY_VALUE_ERROR, spiky_lm_last_error());
    TORCH_CHECK(false, spiky_lm_last_error());
}

int type_code(ScalarType t) {
    return t == at::kFloat ? SPIKY_F32 : t == at::kBFloat16 ? SPIKY_BF16 : t == at::kHalf ? SPIKY_F16 : -1;
}

int type_code(const Tensor &t, const char *name) {
    const int code = type_code(t.scalar_type());
    TORCH_CHECK(code >= 0, "tensor ", name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
    return code;
}

// With its memory's values: torch keeps the sign of imaginary parts of conjugates beside them.
Tensor settled(const Tensor &t) { return t.is_neg() ? t.resolve_neg() : t; }

Tensor device_tensor(PyObject *o, const char *name) {
    TORCH_CHECK(THPVariable_Check(o), "tensor ", name, " must be a torch.Tensor");
    const Tensor &t = THPVariable_Unpack(o);
    TORCH_CHECK(t.device().is_cuda(), "tensor ", name, " must be on CUDA");
    return settled(t);
}

// A trace sees torch's own calls alone, and would keep the results here as constants.
void check_trace() {
    TORCH_CHECK(!at::tracer::impl::is_dispatch_enabled(),
                "spiky_amd's language-model operators cannot be traced by torch.jit.trace");
}

// Forward-mode derivatives are not computed, and a result without a tangent would count as constant.
void check_tangent(PyObject *o, const char *name) {
    TORCH_CHECK_NOT_IMPLEMENTED(!THPVariable_Check(o) || !THPVariable_Unpack(o)._fw_grad(0).defined(),
                                "spiky_amd's language-model operators have no forward-mode derivatives, but tensor ",
                                name, " has a tangent");
}

// Undefined for None.
Tensor device_tensor(PyObject *o, const char *name, c10::Device device) {
    if (o == Py_None) return Tensor();
    Tensor t = device_tensor(o, name);
    TORCH_CHECK(t.device() == device, "tensor ", name, " must be on ", device, ", got ", t.device());
    return t;
}

void *pointer(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

double number(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}

uint64_t bits64(PyObject *o) {
    THPObjectPtr index(PyNumber_Index(o));
    if (!index) throw python_error();
    const uint64_t v = PyLong_AsUnsignedLongLongMask(index.get());
    if (v == (uint64_t)-1 && PyErr_Occurred()) throw python_error();
    return v;
}

double probability(PyObject *o) {
    const double p = number(o);
    TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "dropout probability must be between 0 and 1, got ", p);
    return p;
}

struct Generator {
    uint64_t seed = 0, offset = 0;
    Tensor state;  // [seed, offset] in device memory, in their place
};

Generator generator(PyObject *seed, PyObject *offset, c10::Device device) {
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
std::pair<Tensor, int64_t> as_rows(const Tensor &given) {
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

int64_t rows_of(const Tensor &t) {
    const int64_t cols = t.dim() ? t.size(-1) : 1;
    return cols ? t.numel() / cols : 0;
}

// An uninitialised tensor, without the dispatcher's way to the same call.
Tensor fresh(at::IntArrayRef sizes, ScalarType type, c10::Device device) {
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
void check_capture(const Node &node, c10::Device device) {
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

bool needs_grad(const Tensor &t) { return t.defined() && t.requires_grad(); }

// Gradients of the gradients are not computed: a backward pass through these raises.
struct Twice : Node {
    variable_list apply(variable_list &&) override {
        TORCH_CHECK(false, "spiky_amd's language-model operators cannot be differentiated twice");
    }
};

variable_list once_differentiable(variable_list &&grads, const torch::autograd::edge_list &inputs) {
    if (!at::GradMode::is_enabled()) return std::move(grads);
    auto stop = std::make_shared<Twice>();
    stop->set_next_edges(torch::autograd::edge_list(inputs));  // so that a search for them comes by here
    for (Tensor &t : grads)
        if (t.defined()) torch::autograd::set_history(t, stop);
    return std::move(grads);
}

// ---- dropout ----------------------------------------------------------------
Tensor apply_dropout(const Tensor &given, double p, uint64_t seed, uint64_t offset, const Tensor &state) {
    OnDevice on(given.device());
    auto [x, stride] = as_rows(given);
    Tensor y = fresh(x.sizes(), x.scalar_type(), x.device());
    check(spiky_lm_dropout(x.data_ptr(), stride, y.data_ptr(), rows_of(x), x.dim() ? x.size(-1) : 1,
                           type_code(x, "x"), p, seed, offset, static_cast<const int64_t *>(pointer(state)),
                           on.stream));
    return y;
}

struct CounterDropoutBackward : Node {
    double p;
    uint64_t seed, offset;
    bool has_state;
    SavedVariable state;

    variable_list apply(variable_list &&grads) override {
        if (!grads[0].defined()) return {Tensor()};
        check_capture(*this, grads[0].device());
        at::AutoGradMode off(false);
        const Tensor s = has_state ? state.unpack() : Tensor();
        Tensor dx = apply_dropout(grads[0], p, seed, offset, s);
        return {dx};
    }
    void release_variables() override { state.reset_data(); }
};

// Runs a node's gradients, and marks them where a graph of them is asked for.
template <typename N>
struct Once : N {
    variable_list apply(variable_list &&grads) override {
        return once_differentiable(N::apply(std::move(grads)), N::next_edges());
    }
};

PyObject *dropout(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 4, "dropout takes 4 arguments");
    check_trace();
    check_tangent(args[0], "x");
    const Tensor x = device_tensor(args[0], "x");
    type_code(x, "x");
    const double p = probability(args[1]);
    const Generator g = generator(args[2], args[3], x.device());
    if (!at::GradMode::is_enabled() || !x.requires_grad())
        return THPVariable_Wrap(apply_dropout(x, p, g.seed, g.offset, g.state));
    Tensor y;
    {
        at::AutoGradMode off(false);
        y = apply_dropout(x, p, g.seed, g.offset, g.state);
    }
    auto node = std::make_shared<Once<CounterDropoutBackward>>();
    node->p = p;
    node->seed = g.seed;
    node->offset = g.offset;
    node->has_state = g.state.defined();
    if (node->has_state) node->state = SavedVariable(g.state, false);
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    torch::autograd::set_history(y, node);
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// ---- residual join ----------------------------------------------------------
// What a call has beside its tensors.
struct How {
    int post, pre;
    double post_eps, pre_eps, alpha, beta, p;
    uint64_t seed, offset;
    int64_t gate_rows;
    ScalarType dtype;  // of the branch
};

// residual, branch, post weight and bias, gate, pre weight and bias
enum { kRes, kBranch, kPostWeight, kPostBias, kGate, kPreWeight, kPreBias, kInputs };
typedef std::array<Tensor, kInputs> Inputs;

// The C arguments; res and branch keep what they point to.
spiky_lm_residual_args join_args(const How &how, const Inputs &in, const Tensor &state, const Tensor &stats,
                                 Tensor &res, Tensor &branch) {
    spiky_lm_residual_args a = {};
    std::tie(res, a.residual_stride) = as_rows(in[kRes]);
    if (in[kBranch].defined()) std::tie(branch, a.branch_stride) = as_rows(in[kBranch]);
    a.rows = rows_of(res);
    a.cols = res.size(-1);
    a.res_dtype = type_code(res.scalar_type());
    a.act_dtype = type_code(how.dtype);
    a.post_norm = how.post;
    a.pre_norm = how.pre;
    for (int i : {kPostWeight, kPostBias, kPreWeight, kPreBias})
        if (in[i].defined()) a.par_f32 = in[i].scalar_type() == at::kFloat;
    a.gate_f32 = in[kGate].defined() && in[kGate].scalar_type() == at::kFloat;
    a.residual = pointer(res);
    a.branch = pointer(branch);
    a.post_weight = pointer(in[kPostWeight]);
    a.post_bias = pointer(in[kPostBias]);
    a.pre_weight = pointer(in[kPreWeight]);
    a.pre_bias = pointer(in[kPreBias]);
    a.gate = pointer(in[kGate]);
    a.gate_rows = how.gate_rows;
    a.post_eps = how.post_eps;
    a.pre_eps = how.pre_eps;
    a.residual_scale = how.alpha;
    a.branch_scale = how.beta;
    a.dropout_p = how.p;
    a.seed = how.seed;
    a.offset = how.offset;
    a.rng = static_cast<const int64_t *>(pointer(state));
    a.stats = static_cast<float *>(pointer(stats));
    return a;
}

// (stream, normed), undefined where there is none.
std::pair<Tensor, Tensor> join_forward(const How &how, const Inputs &in, const Tensor &state, const Tensor &stats) {
    OnDevice on(in[kRes].device());
    Tensor res, branch, out, normed;
    const spiky_lm_residual_args a = join_args(how, in, state, stats, res, branch);
    if (branch.defined()) out = fresh(res.sizes(), res.scalar_type(), res.device());
    if (how.pre) normed = fresh(res.sizes(), how.dtype, res.device());
    check(spiky_lm_residual_norm(&a, pointer(out), pointer(normed), on.stream));
    return {out, normed};
}

struct ResidualNormBackward : Node {
    How how;
    bool has_state = false, has[kInputs] = {};
    SavedVariable state, saved[kInputs];
    Tensor stats;

    variable_list apply(variable_list &&grads) override {
        variable_list out(kInputs);
        Tensor d_out = grads[0], d_normed = grads[1];
        if (!d_out.defined() && !d_normed.defined()) return out;
        at::AutoGradMode off(false);
        Inputs in;
        for (int i = 0; i < kInputs; i++)
            if (has[i]) in[i] = saved[i].unpack();
        const Tensor rng = has_state ? state.unpack() : Tensor();
        TORCH_CHECK(stats.defined(), torch::autograd::ERR_BACKWARD_TWICE);
        check_capture(*this, in[kRes].device());
        OnDevice on(in[kRes].device());
        Tensor res, branch;
        const spiky_lm_residual_args a = join_args(how, in, rng, stats, res, branch);
        // parameters of a pre norm whose output has no gradient get none written
        const bool idle = !d_normed.defined();
        spiky_lm_residual_grads g = {};
        for (int i = 0; i < kInputs; i++) {
            if (!has[i] || !task_should_compute_output(i)) continue;
            const bool zero = a.rows == 0 || a.cols == 0 || (idle && (i == kPreWeight || i == kPreBias));
            out[i] = zero ? at::zeros(in[i].sizes(), in[i].options().requires_grad(false))
                          : fresh(in[i].sizes(), in[i].scalar_type(), in[i].device());
        }
        if (d_out.defined()) std::tie(d_out, g.d_out_stride) = as_rows(d_out);
        if (d_normed.defined()) std::tie(d_normed, g.d_normed_stride) = as_rows(d_normed);
        g.d_out = pointer(d_out);
        g.d_normed = pointer(d_normed);
        g.d_residual = pointer(out[kRes]);
        g.d_branch = pointer(out[kBranch]);
        g.d_post_weight = pointer(out[kPostWeight]);
        g.d_post_bias = pointer(out[kPostBias]);
        g.d_gate = pointer(out[kGate]);
        g.d_pre_weight = idle ? nullptr : pointer(out[kPreWeight]);
        g.d_pre_bias = idle ? nullptr : pointer(out[kPreBias]);
        g.workspace_bytes = spiky_lm_residual_norm_workspace(&a, &g);
        Tensor workspace = fresh({(int64_t)g.workspace_bytes}, at::kByte, res.device());
        g.workspace = workspace.data_ptr();
        check(spiky_lm_residual_norm_backward(&a, &g, on.stream));
        return out;
    }
    void release_variables() override {
        state.reset_data();
        for (SavedVariable &s : saved) s.reset_data();
        stats.reset();
    }
};

int norm_kind(PyObject *norm, PyObject *weight, PyObject *bias, const char *name) {
    if (norm == Py_None) {
        TORCH_CHECK_VALUE(weight == Py_None && bias == Py_None, name, "_weight and ", name, "_bias need a ", name,
                          "_norm");
        return SPIKY_NORM_NONE;
    }
    if (PyUnicode_Check(norm)) {
        if (PyUnicode_CompareWithASCIIString(norm, "rms") == 0) return SPIKY_NORM_RMS;
        if (PyUnicode_CompareWithASCIIString(norm, "layer") == 0) return SPIKY_NORM_LAYER;
    }
    TORCH_CHECK_VALUE(false, name, "_norm must be None, 'rms' or 'layer'");
}

// The gate, and the consecutive rows that share one of its rows.  Gates that are
// one row, one row for each index of some leading dimensions, or of the full shape
// are read as they are; others that broadcast to the shape are expanded to it.
std::pair<Tensor, int64_t> gate_rows(const Tensor &gate, at::IntArrayRef shape) {
    const int64_t dim = (int64_t)shape.size(), missing = dim - gate.dim();
    auto lead = [&](int64_t k) { return k < missing ? (int64_t)1 : gate.size(k - missing); };
    bool fits = missing >= 0;
    for (int64_t k = 0; fits && k < dim; k++) fits = lead(k) == 1 || lead(k) == shape[k];
    TORCH_CHECK_VALUE(fits, "gate of shape ", gate.sizes(), " does not broadcast to ", shape);
    int64_t k = dim - 1;
    while (k > 0 && lead(k - 1) == 1) k--;
    bool as_is = lead(dim - 1) == shape[dim - 1];
    for (int64_t i = 0; i < k; i++) as_is = as_is && lead(i) == shape[i];
    if (!as_is) return {gate.expand(shape).contiguous(), 1};
    int64_t share = 1;
    for (int64_t i = k; i < dim - 1; i++) share *= shape[i];
    return {gate.contiguous(), std::max<int64_t>(share, 1)};
}

PyObject *pair(PyObject *first, PyObject *second) {
    PyObject *t = PyTuple_New(2);
    if (!t) throw python_error();
    PyTuple_SET_ITEM(t, 0, first);
    PyTuple_SET_ITEM(t, 1, second);
    return t;
}

PyObject *wrapped(const Tensor &t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_INCREF(Py_None);
    return Py_None;
}

PyObject *residual_norm(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 17, "residual_norm takes 17 arguments");
    check_trace();
    enum {
        Residual, Branch, PostNorm, PostWeight, PostBias, PostEps, Gate, ResidualScale, BranchScale, DropoutP, Seed,
        Offset, PreNorm, PreWeight, PreBias, PreEps, Dtype
    };
    const std::pair<int, const char *> differentiable[] = {
        {Residual, "residual"}, {Branch, "branch"},         {PostWeight, "post_weight"}, {PostBias, "post_bias"},
        {Gate, "gate"},         {PreWeight, "pre_weight"}, {PreBias, "pre_bias"},
    };
    for (const auto &[arg, name] : differentiable) check_tangent(args[arg], name);
    Inputs in;
    in[kRes] = device_tensor(args[Residual], "residual");
    const Tensor &res = in[kRes];
    const int res_code = type_code(res, "residual");
    TORCH_CHECK_VALUE(res.dim() > 0, "residual must have at least one dimension");
    const c10::Device device = res.device();
    How how;
    how.post = norm_kind(args[PostNorm], args[PostWeight], args[PostBias], "post");
    how.pre = norm_kind(args[PreNorm], args[PreWeight], args[PreBias], "pre");
    how.alpha = number(args[ResidualScale]);
    how.beta = number(args[BranchScale]);
    how.p = probability(args[DropoutP]);
    how.post_eps = number(args[PostEps]);
    how.pre_eps = number(args[PreEps]);
    std::optional<ScalarType> dtype;
    if (args[Dtype] != Py_None) {
        TORCH_CHECK(THPDtype_Check(args[Dtype]), "dtype must be a torch.dtype");
        dtype = reinterpret_cast<THPDtype *>(args[Dtype])->scalar_type;
    }
    in[kBranch] = device_tensor(args[Branch], "branch", device);
    if (!in[kBranch].defined()) {
        TORCH_CHECK_VALUE(how.post == SPIKY_NORM_NONE && args[Gate] == Py_None && how.p == 0.0 && how.alpha == 1.0,
                          "a post_norm, gate, dropout or scale needs a branch");
        TORCH_CHECK_VALUE(how.pre != SPIKY_NORM_NONE, "neither a branch nor a pre_norm");
        how.dtype = dtype.value_or(res.scalar_type());
    } else {
        type_code(in[kBranch], "branch");
        TORCH_CHECK_VALUE(in[kBranch].sizes() == res.sizes(), "branch of shape ", in[kBranch].sizes(),
                          " for a residual of ", res.sizes());
        how.dtype = in[kBranch].scalar_type();
        TORCH_CHECK_VALUE(!dtype || *dtype == how.dtype, "dtype is the branch's where there is one");
    }
    TORCH_CHECK(type_code(how.dtype) >= 0 && (res_code == type_code(how.dtype) || res_code == SPIKY_F32),
                "a residual of ", res.scalar_type(), " does not go with a branch of ", how.dtype);
    const std::pair<int, std::pair<int, const char *>> parameters[] = {
        {kPostWeight, {PostWeight, "post_weight"}},
        {kPostBias, {PostBias, "post_bias"}},
        {kPreWeight, {PreWeight, "pre_weight"}},
        {kPreBias, {PreBias, "pre_bias"}},
    };
    std::optional<ScalarType> common;
    for (const auto &[i, from] : parameters) {
        const auto &[arg, name] = from;
        const Tensor t = device_tensor(args[arg], name, device);
        if (!t.defined()) continue;
        TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == res.size(-1), name, " must have shape (", res.size(-1),
                          ",), got ", t.sizes());
        TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == how.dtype, "tensor ", name,
                    " must be float32 or ", how.dtype, ", got ", t.scalar_type());
        TORCH_CHECK(!common || *common == t.scalar_type(), "the norms' parameters must have one type");
        common = t.scalar_type();
        in[i] = t.contiguous();
    }
    how.gate_rows = 1;
    if (args[Gate] != Py_None) {
        const Tensor gate = device_tensor(args[Gate], "gate", device);
        TORCH_CHECK(gate.scalar_type() == at::kFloat || gate.scalar_type() == how.dtype,
                    "tensor gate must be float32 or ", how.dtype, ", got ", gate.scalar_type());
        std::tie(in[kGate], how.gate_rows) = gate_rows(gate, res.sizes());
    }
    Generator g;
    if (how.p > 0.0) g = generator(args[Seed], args[Offset], device);
    how.seed = g.seed;
    how.offset = g.offset;

    bool train = false;
    for (const Tensor &t : in) train = train || needs_grad(t);
    std::pair<Tensor, Tensor> result;
    if (!train || !at::GradMode::is_enabled()) {
        result = join_forward(how, in, g.state, Tensor());
    } else {
        auto node = std::make_shared<Once<ResidualNormBackward>>();
        {
            at::AutoGradMode off(false);
            node->stats = fresh({rows_of(res), 4}, at::kFloat, device);
            result = join_forward(how, in, g.state, node->stats);
        }
        node->how = how;
        node->has_state = g.state.defined();
        if (node->has_state) node->state = SavedVariable(g.state, false);
        for (int i = 0; i < kInputs; i++) {
            node->has[i] = in[i].defined();
            if (node->has[i]) node->saved[i] = SavedVariable(in[i], false);
        }
        node->set_next_edges(torch::autograd::collect_next_edges(in[0], in[1], in[2], in[3], in[4], in[5], in[6]));
        torch::autograd::set_history(result.first, node);
        torch::autograd::set_history(result.second, node);
    }
    if (in[kBranch].defined()) return pair(THPVariable_Wrap(result.first), wrapped(result.second));
    Py_INCREF(args[Residual]);
    return pair(args[Residual], wrapped(result.second));
    END_HANDLE_TH_ERRORS
}

// ---- logits -----------------------------------------------------------------
// n rows of `width` bytes in memory, `step` bytes apart.
struct Span {
    uintptr_t at = 0;
    int64_t n = 0, step = 0, width = 0;
};

// The rows of a tensor with contiguous columns, `stride` elements apart; one row for all where that is 0.
Span span_of(const Tensor &t, int64_t stride) {
    if (!t.defined() || t.numel() == 0) return {};
    const int64_t size = (int64_t)t.element_size(), rows = t.dim() == 2 ? t.size(0) : 1;
    return {reinterpret_cast<uintptr_t>(t.data_ptr()), stride ? rows : 1, stride * size, t.size(-1) * size};
}

// Rows of both are in the order of their addresses, so one walk along them meets any two that overlap.
bool overlap(const Span &a, const Span &b) {
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

bool is_index(const Tensor &t, const char *name) {
    const bool wide = t.scalar_type() == at::kLong;
    TORCH_CHECK(wide || t.scalar_type() == at::kInt, "tensor ", name, " must have dtype int32 or int64, got ",
                t.scalar_type());
    return wide;
}

// [n] for every row, or [rows, n]: with contiguous columns, and the distance of its rows.
std::pair<Tensor, int64_t> by_row(const Tensor &t, const char *name, int64_t rows) {
    TORCH_CHECK_VALUE(t.dim() == 1 || (t.dim() == 2 && t.size(0) == rows), name, " must be [n] or [", rows,
                      ", n], got ", t.sizes());
    if (t.dim() == 1) return {t.contiguous(), 0};
    Tensor c = t.size(1) > 1 && t.stride(1) != 1 ? t.contiguous() : t;
    const int64_t stride = c.stride(0);
    return {c, stride};
}

PyObject *process_logits(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 14, "process_logits takes 14 arguments");
    check_trace();
    enum {
        Logits, TokenIds, Lengths, PromptLengths, Repetition, Presence, Frequency, Bias, BiasIds, BiasValues,
        Temperature, Mask, Out, Dtype
    };
    Tensor logits = device_tensor(args[Logits], "logits");
    spiky_lm_logits_args a = {};
    a.dtype = type_code(logits, "logits");
    const c10::Device device = logits.device();
    TORCH_CHECK_VALUE(logits.dim() == 2, "logits must be [B, V], got ", logits.sizes());
    const int64_t rows = logits.size(0), vocab = logits.size(1);
    at::AutoGradMode off(false);
    OnDevice on(device);
    if (vocab > 1 && logits.stride(1) != 1) {
        TORCH_CHECK_VALUE(args[Out] != args[Logits], "logits that are written in place need contiguous columns");
        logits = logits.contiguous();
    }
    std::optional<ScalarType> dtype;
    if (args[Dtype] != Py_None) {
        TORCH_CHECK(THPDtype_Check(args[Dtype]), "dtype must be a torch.dtype");
        dtype = reinterpret_cast<THPDtype *>(args[Dtype])->scalar_type;
    }
    auto fits = [&](ScalarType t) { return t == logits.scalar_type() || t == at::kFloat; };
    TORCH_CHECK_VALUE(!THPVariable_Check(args[Out]) || !THPVariable_Unpack(args[Out]).is_neg(),
                      "out must hold its values' signs");
    Tensor out = device_tensor(args[Out], "out", device);
    if (!out.defined()) {
        const ScalarType t = dtype.value_or(logits.scalar_type());
        TORCH_CHECK_VALUE(fits(t), "dtype must be ", logits.scalar_type(), " or float32, got ", t);
        out = fresh({rows, vocab}, t, device);
    } else {
        TORCH_CHECK_VALUE(out.sizes() == logits.sizes() && fits(out.scalar_type()) &&
                              (!dtype || *dtype == out.scalar_type()),
                          "out must be ", logits.sizes(), " of ", logits.scalar_type(), " or float32, or of dtype");
        TORCH_CHECK_VALUE(vocab <= 1 || out.stride(1) == 1, "out must have contiguous columns");
        TORCH_CHECK_VALUE(rows <= 1 || out.stride(0) >= vocab, "the rows of out must not overlap");
        TORCH_CHECK_VALUE(out.data_ptr() != logits.data_ptr() ||
                              (out.scalar_type() == logits.scalar_type() &&
                               (rows <= 1 || out.stride(0) == logits.stride(0))),
                          "out may be logits, but not another view of them");
        TORCH_CHECK_VALUE(!out.requires_grad(), "out must not require a gradient");
    }
    a.rows = rows;
    a.vocab = vocab;
    a.logits = logits.data_ptr();
    a.logits_stride = logits.stride(0);
    a.out = out.data_ptr();
    a.out_stride = out.stride(0);
    a.out_dtype = type_code(out.scalar_type());

    Tensor tokens = device_tensor(args[TokenIds], "tokens", device), lengths, prompts;
    if (tokens.defined()) {
        TORCH_CHECK_VALUE(tokens.dim() == 2, "tokens must be [", rows, ", L], got ", tokens.sizes());
        a.tokens_i64 = is_index(tokens, "tokens");
        std::tie(tokens, a.tokens_stride) = by_row(tokens, "tokens", rows);
        a.history = tokens.size(1);
        a.tokens = a.history ? tokens.data_ptr() : nullptr;
        auto length_of = [&](int arg, const char *name) {
            Tensor t = device_tensor(args[arg], name, device);
            if (!t.defined()) return t;
            is_index(t, name);
            TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == rows, name, " must have shape (", rows, ",), got ",
                              t.sizes());
            return t.contiguous();
        };
        lengths = length_of(Lengths, "lengths");
        prompts = length_of(PromptLengths, "prompt_lengths");
        if (lengths.defined() && prompts.defined() && prompts.scalar_type() != lengths.scalar_type()) {
            // a prompt past 32 bits is past any history: both go as int64
            lengths = lengths.to(at::kLong);
            prompts = prompts.to(at::kLong);
        }
        const Tensor &either = lengths.defined() ? lengths : prompts;
        a.lengths_i64 = either.defined() && either.scalar_type() == at::kLong;
        a.lengths = pointer(lengths);
        a.prompt_lengths = pointer(prompts);
    } else {
        TORCH_CHECK_VALUE(args[Lengths] == Py_None && args[PromptLengths] == Py_None, "lengths need tokens");
    }

    // one value for all rows, or a float32 tensor of one for each
    auto setting = [&](int arg, const char *name, float &value, const float *&values) {
        Tensor t;
        if (!THPVariable_Check(args[arg])) {
            value = (float)number(args[arg]);
            return t;
        }
        t = device_tensor(args[arg], name, device);
        TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == rows, name, " must be a number or have shape (", rows,
                          ",), got ", t.sizes());
        TORCH_CHECK(t.is_floating_point(), "tensor ", name, " must be floating point, got ", t.scalar_type());
        t = t.to(at::kFloat).contiguous();
        values = t.data_ptr<float>();
        value = 1.f;
        return t;
    };
    const Tensor repetition = setting(Repetition, "repetition_penalty", a.repetition, a.repetition_rows);
    TORCH_CHECK_VALUE(repetition.defined() || a.repetition > 0.f, "repetition_penalty must be positive, got ",
                      a.repetition);
    const Tensor presence = setting(Presence, "presence_penalty", a.presence, a.presence_rows);
    const Tensor frequency = setting(Frequency, "frequency_penalty", a.frequency, a.frequency_rows);
    const Tensor temperature = setting(Temperature, "temperature", a.temperature, a.temperature_rows);

    Tensor bias = device_tensor(args[Bias], "bias", device);
    if (bias.defined()) {
        a.bias_dtype = type_code(bias, "bias");
        std::tie(bias, a.bias_stride) = by_row(bias, "bias", rows);
        TORCH_CHECK_VALUE(bias.size(-1) == vocab, "bias must be [", vocab, "] or [", rows, ", ", vocab, "], got ",
                          bias.sizes());
        a.bias = bias.data_ptr();
    }
    TORCH_CHECK_VALUE((args[BiasIds] == Py_None) == (args[BiasValues] == Py_None),
                      "bias_ids and bias_values go together");
    Tensor ids = device_tensor(args[BiasIds], "bias_ids", device);
    Tensor values = device_tensor(args[BiasValues], "bias_values", device);
    if (ids.defined()) {
        a.bias_ids_i64 = is_index(ids, "bias_ids");
        TORCH_CHECK_VALUE(values.sizes() == ids.sizes(), "bias_values must have the shape of bias_ids, ", ids.sizes());
        TORCH_CHECK(values.scalar_type() == at::kFloat, "tensor bias_values must be float32, got ",
                    values.scalar_type());
        std::tie(ids, a.bias_ids_stride) = by_row(ids, "bias_ids", rows);
        std::tie(values, a.bias_values_stride) = by_row(values, "bias_values", rows);
        a.n_bias = ids.size(-1);
        if (a.n_bias) {
            a.bias_ids = ids.data_ptr();
            a.bias_values = values.data_ptr<float>();
        }
    }
    Tensor mask = device_tensor(args[Mask], "mask", device);
    if (mask.defined()) {
        TORCH_CHECK(mask.scalar_type() == at::kBool || mask.scalar_type() == at::kInt,
                    "tensor mask must have dtype bool or int32, got ", mask.scalar_type());
        a.mask_bits = mask.scalar_type() == at::kInt;
        std::tie(mask, a.mask_stride) = by_row(mask, "mask", rows);
        const int64_t need = a.mask_bits ? (vocab + 31) / 32 : vocab;
        TORCH_CHECK_VALUE(mask.size(-1) == need, "mask must be [", need, "] or [", rows, ", ", need, "], got ",
                          mask.sizes());
        a.mask = mask.data_ptr();
    }
    if (args[Out] == Py_None) {
        check(spiky_lm_process_logits(&a, on.stream));
        return THPVariable_Wrap(out);
    }
    // Workgroups read the row's settings, tokens and biases at any time, and other elements of the rest than
    // they write.  Logits, or a bias, in the very place of the result are read by the lane that writes there.
    const Span to = span_of(out, a.out_stride);
    auto apart = [&](const Tensor &t, int64_t stride, const char *name, bool by_element = false) {
        const Span from = span_of(t, stride);
        const bool in_place = by_element && from.at == to.at && from.width == to.width && from.n == to.n &&
                              (to.n == 1 || from.step == to.step);
        TORCH_CHECK_VALUE(in_place || !overlap(from, to), "out must not overlap ", name);
    };
    apart(logits, a.logits_stride, "logits other than as the same tensor", true);
    apart(bias, a.bias_stride, "bias", true);
    apart(mask, a.mask_stride, "mask");
    apart(tokens, a.tokens_stride, "tokens");
    apart(ids, a.bias_ids_stride, "bias_ids");
    apart(values, a.bias_values_stride, "bias_values");
    const std::pair<const Tensor &, const char *> by_rows[] = {
        {lengths, "lengths"},
        {prompts, "prompt_lengths"},
        {repetition, "repetition_penalty"},
        {presence, "presence_penalty"},
        {frequency, "frequency_penalty"},
        {temperature, "temperature"},
    };
    for (const auto &[t, name] : by_rows) apart(t, 0, name);
    check(spiky_lm_process_logits(&a, on.stream));
    if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
    Py_INCREF(args[Out]);
    return args[Out];
    END_HANDLE_TH_ERRORS
}

// ---- for tests --------------------------------------------------------------
PyObject *rows_of_tensor(PyObject *, PyObject *o) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(THPVariable_Check(o), "not a torch.Tensor");
    auto [t, stride] = as_rows(THPVariable_Unpack(o));
    return pair(THPVariable_Wrap(t), PyLong_FromLongLong(stride));
    END_HANDLE_TH_ERRORS
}

PyObject *rows_of_gate(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 2 && THPVariable_Check(args[0]) && THPVariable_Check(args[1]), "a gate and a branch");
    auto [t, share] = gate_rows(THPVariable_Unpack(args[0]), THPVariable_Unpack(args[1]).sizes());
    return pair(THPVariable_Wrap(t), PyLong_FromLongLong(share));
    END_HANDLE_TH_ERRORS
}

PyObject *rows_overlap(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 2 && THPVariable_Check(args[0]) && THPVariable_Check(args[1]), "two tensors of rows");
    const Tensor &a = THPVariable_Unpack(args[0]), &b = THPVariable_Unpack(args[1]);
    return PyBool_FromLong(overlap(span_of(a, a.stride(0)), span_of(b, b.stride(0))));
    END_HANDLE_TH_ERRORS
}

template <typename F>
PyCFunction fast(F *f) {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {
    {"dropout", fast(dropout), METH_FASTCALL, "x, p, seed, offset"},
    {"residual_norm", fast(residual_norm), METH_FASTCALL, "the arguments of spiky_amd.residual_norm, in its order"},
    {"process_logits", fast(process_logits), METH_FASTCALL, "the arguments of spiky_amd.process_logits, in its order"},
    {"rows_of_tensor", rows_of_tensor, METH_O, "the tensor as rows of its last dimension, and their distance"},
    {"rows_of_gate", fast(rows_of_gate), METH_FASTCALL, "the gate as read for a branch, and the rows that share one"},
    {"rows_overlap", fast(rows_overlap), METH_FASTCALL, "whether rows of two matrices share memory"},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_lm_torch", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__lm_torch(void) { return PyModule_Create(&module); }
