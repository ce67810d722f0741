// lm_tokens_torch.cpp -- the operators of include/spiky_lm_tokens.h on torch tensors.
// Host code only; all device work goes through the C ABI of libspiky_lut.so.
#include <algorithm>
#include <cmath>
#include <functional>
#include <numeric>
#include <vector>

#include "lm_torch.h"

namespace lm_torch {
namespace {

// ---- embedding ----------------------------------------------------------------
// The C arguments but for the weight.
spiky_lm_embed_args embed_args(const Tensor &tokens, at::IntArrayRef table, ScalarType weight, ScalarType out,
                               double scale) {
    spiky_lm_embed_args a = {};
    a.n = tokens.numel();
    a.vocab = table[0];
    a.cols = table[1];
    a.tokens_i64 = tokens.scalar_type() == at::kLong;
    a.weight_dtype = type_code(weight);
    a.out_dtype = type_code(out);
    a.tokens = pointer(tokens);
    a.weight_stride = table[1];
    a.scale = scale;
    return a;
}

Tensor lookup(const Tensor &tokens, const Tensor &weight, ScalarType dtype, double scale) {
    OnDevice on(weight.device());
    auto [table, stride] = as_rows(weight);
    spiky_lm_embed_args a = embed_args(tokens, table.sizes(), table.scalar_type(), dtype, scale);
    a.weight = pointer(table);
    a.weight_stride = stride;
    std::vector<int64_t> shape(tokens.sizes().begin(), tokens.sizes().end());
    shape.push_back(weight.size(1));
    Tensor out = fresh(shape, dtype, weight.device());
    check(spiky_lm_embed(&a, out.data_ptr(), on.stream));
    return out;
}

struct EmbedTokensBackward : Node {
    SavedVariable tokens;
    int64_t table[2];
    ScalarType weight, dtype;
    double scale;

    variable_list apply(variable_list &&grads) override {
        if (!grads[0].defined()) return {Tensor()};
        at::AutoGradMode off(false);
        const Tensor t = tokens.unpack();
        const c10::Device device = grads[0].device();
        check_capture(*this, device);
        OnDevice on(device);
        const spiky_lm_embed_args a = embed_args(t, table, weight, dtype, scale);
        auto [d_out, stride] = as_rows(grads[0]);
        Tensor d_weight = fresh(table, weight, device);
        const uint64_t bytes = spiky_lm_embed_workspace(&a);
        Tensor workspace = fresh({(int64_t)bytes}, at::kByte, device);
        check(spiky_lm_embed_backward(&a, d_out.data_ptr(), stride, d_weight.data_ptr(), workspace.data_ptr(), bytes,
                                      on.stream));
        return {d_weight};
    }
    void release_variables() override { tokens.reset_data(); }
};

// A tensor [searches, beams] of whole numbers or truth values.
Tensor by_beam(PyObject *o, const char *name, at::IntArrayRef shape, c10::Device device) {
    Tensor t = device_tensor(o, name, device);
    if (!t.defined()) return t;
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape ", shape, ", got ", t.sizes());
    return t.contiguous();
}

PyObject *triple(const Tensor &a, const Tensor &b, const Tensor &c) {
    PyObject *t = PyTuple_New(3);
    if (!t) throw python_error();
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(a));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(b));
    PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(c));
    return t;
}

// ---- reordering -----------------------------------------------------------------
// One side of a state: bytes from search to search, beam to beam and run to run.
struct Side {
    uintptr_t at = 0;
    int64_t search = 0, beam = 0, run = 0;
    uint64_t runs = 1, run_bytes = 0;
};

// The dimensions behind the first two, joined from the last on while they lie behind one another:
// false where more than one dimension is left beside the contiguous one.
bool side_of(const Tensor &t, Side &s) {
    const int64_t size = (int64_t)t.element_size();
    s.at = reinterpret_cast<uintptr_t>(t.data_ptr());
    s.search = t.stride(0) * size;
    s.beam = t.stride(1) * size;
    int64_t bytes = size, k = t.dim() - 1;
    for (; k >= 2 && (t.size(k) == 1 || t.stride(k) * size == bytes); k--) bytes *= t.size(k);
    s.run_bytes = bytes;
    s.runs = 1;
    s.run = 0;
    for (; k >= 2; k--) {
        if (t.size(k) == 1) continue;
        if (s.run == 0 && s.runs == 1)
            s.run = t.stride(k) * size;
        else if (t.stride(k) * size != s.run * (int64_t)s.runs)
            return false;
        s.runs *= t.size(k);
    }
    return true;
}

// A side's bytes: the steps of its dimensions of more than one index, from the largest on, and their numbers of indexes.
struct Bytes {
    uintptr_t at = 0, end = 0;  // the first byte, and the first past it
    int64_t run = 0;
    std::pair<int64_t, int64_t> steps[3];
    int n = 0;
    int64_t unit = 0;       // all steps are multiples of it
    bool expanded = false;  // a dimension's indexes are all at one place

    Bytes(const Side &s, int64_t searches, int64_t beams) : at(s.at), run((int64_t)s.run_bytes) {
        for (const auto &[step, many] :
             {std::pair<int64_t, int64_t>{s.search, searches}, {s.beam, beams}, {s.run, (int64_t)s.runs}}) {
            if (many <= 1) continue;
            if (step == 0) {
                expanded = true;
                continue;
            }
            steps[n++] = {step, many};
            unit = std::gcd(unit, step);
        }
        std::sort(steps, steps + n, std::greater<>());
        end = at + s.run_bytes;
        for (int i = 0; i < n; i++) end += steps[i].first * (steps[i].second - 1);
    }
};

// No byte is there twice: each stride reaches past what the smaller ones span.
bool once_each(const Bytes &b) {
    int64_t span = b.run;
    for (int i = b.n - 1; i >= 0; i--) {
        if (b.steps[i].first < span) return false;
        span += b.steps[i].first * (b.steps[i].second - 1);
    }
    return !b.expanded;
}

// Whether two sides share a byte: `d` bytes from a's first to b's first, and for each its steps from the largest
// on and its run's bytes.  Steps that both have are taken together, as only the difference of the indexes counts; else
// the larger step goes index by index, `left` of them in all: past that, they are taken to share one.
struct Steps {
    const std::pair<int64_t, int64_t> *first, *last;
    int64_t bytes;

    int64_t span() const {
        int64_t span = bytes;
        for (auto s = first; s != last; s++) span += s->first * (s->second - 1);
        return span;
    }
    Steps inner() const { return {first + 1, last, bytes}; }
};

bool meet(int64_t d, const Steps &a, const Steps &b, int &left) {
    if (d >= a.span() || -d >= b.span()) return false;
    if (a.first == a.last && b.first == b.last) return true;
    const int64_t of_a = a.first == a.last ? 0 : a.first->first, of_b = b.first == b.last ? 0 : b.first->first;
    const Steps in_a = of_a >= of_b ? a.inner() : a, in_b = of_b >= of_a ? b.inner() : b;
    const int64_t step = std::max(of_a, of_b);
    // the indexes of b minus a's for which the inner parts' spans meet: -in_b.span() < d + i * step < in_a.span()
    const auto below = [&](int64_t x) { return x >= 0 ? x / step : -((-x + step - 1) / step); };
    const int64_t from = std::max(of_a >= of_b ? 1 - a.first->second : 0, below(-in_b.span() - d) + 1);
    const int64_t to = std::min(of_b >= of_a ? b.first->second - 1 : 0, -below(d - in_a.span()) - 1);
    for (int64_t i = from; i <= to; i++)
        if (left-- <= 0 || meet(d + i * step, in_a, in_b, left)) return true;
    return false;
}

// Sides that share no byte, as the keys and values of one cache: one ends before the other, or all strides of both
// are multiples of one number within which they take different parts, or no two of their runs meet.
bool apart(const Bytes &a, const Bytes &b) {
    if (a.end <= b.at || b.end <= a.at) return true;
    const int64_t distance = (int64_t)(b.at - a.at), unit = std::gcd(a.unit, b.unit);
    if (unit > 0) {
        const int64_t shift = (distance % unit + unit) % unit;
        if (a.run <= shift && shift + b.run <= unit) return true;
    }
    int left = 1 << 14;
    return !meet(distance, {a.steps, a.steps + a.n, a.run}, {b.steps, b.steps + b.n, b.run}, left);
}

// The tensors of a list, a tuple or one tensor.
std::vector<PyObject *> each_of(PyObject *o, bool &one) {
    one = THPVariable_Check(o);
    if (one) return {o};
    TORCH_CHECK(PyList_Check(o) || PyTuple_Check(o), "states must be a torch.Tensor or a list or tuple of them");
    std::vector<PyObject *> items;
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(o); i++) items.push_back(PySequence_Fast_GET_ITEM(o, i));
    return items;
}

}  // namespace

PyObject *embed_tokens(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 4, "embed_tokens takes 4 arguments");
    check_trace();
    enum { Tokens, Weight, Scale, Dtype };
    check_tangent(args[Weight], "weight");
    const Tensor weight = device_tensor(args[Weight], "weight");
    type_code(weight, "weight");
    TORCH_CHECK_VALUE(weight.dim() == 2, "weight must be [V, E], got ", weight.sizes());
    TORCH_CHECK(args[Tokens] != Py_None, "tensor tokens must be a torch.Tensor");
    const Tensor given = device_tensor(args[Tokens], "tokens", weight.device());
    is_index(given, "tokens");
    const double scale = number(args[Scale]);
    TORCH_CHECK_VALUE(std::isfinite((float)scale), "scale must be finite in 32 bits, got ", scale);
    ScalarType dtype = weight.scalar_type();
    if (args[Dtype] != Py_None) {
        TORCH_CHECK(THPDtype_Check(args[Dtype]), "dtype must be a torch.dtype");
        dtype = reinterpret_cast<THPDtype *>(args[Dtype])->scalar_type;
        TORCH_CHECK_VALUE(type_code(dtype) >= 0 && (dtype == weight.scalar_type() || dtype == at::kFloat ||
                                                    weight.scalar_type() == at::kFloat),
                          "dtype must be ", weight.scalar_type(), " or float32, or the weight float32; got ", dtype);
    }
    Tensor y, tokens;
    {
        at::AutoGradMode off(false);
        tokens = given.contiguous();
        y = lookup(tokens, weight, dtype, scale);
    }
    if (!at::GradMode::is_enabled() || !weight.requires_grad()) return THPVariable_Wrap(y);
    auto node = std::make_shared<Once<EmbedTokensBackward>>();
    node->tokens = SavedVariable(tokens, false);
    node->table[0] = weight.size(0);
    node->table[1] = weight.size(1);
    node->weight = weight.scalar_type();
    node->dtype = dtype;
    node->scale = scale;
    node->set_next_edges(torch::autograd::collect_next_edges(weight));
    torch::autograd::set_history(y, node);
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

PyObject *beam_select(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 7, "beam_select takes 7 arguments");
    check_trace();
    enum { Logits, Scores, N, Finished, Pad, Lengths, LengthPenalty };
    check_tangent(args[Logits], "logits");
    check_tangent(args[Scores], "scores");
    at::AutoGradMode off(false);
    Tensor logits = device_tensor(args[Logits], "logits");
    spiky_lm_beams_args a = {};
    a.dtype = type_code(logits, "logits");
    TORCH_CHECK_VALUE(logits.dim() == 3, "logits must be [B, K, V], got ", logits.sizes());
    const c10::Device device = logits.device();
    const int64_t searches = logits.size(0), beams = logits.size(1), vocab = logits.size(2);
    OnDevice on(device);
    if (vocab > 1 && logits.stride(2) != 1) logits = logits.contiguous();
    const int64_t shape[2] = {searches, beams};
    TORCH_CHECK(args[Scores] != Py_None, "tensor scores must be a torch.Tensor");
    const Tensor scores = by_beam(args[Scores], "scores", shape, device);
    TORCH_CHECK(scores.scalar_type() == at::kFloat, "tensor scores must be float32, got ", scores.scalar_type());
    int64_t count = beams;
    if (args[N] != Py_None) count = whole(args[N], "n");
    TORCH_CHECK_VALUE(beams >= 1 && beams <= 64 && count >= 1 && count <= 64, "beams and n must be 1 to 64, got ",
                      beams, " and ", count);
    const Tensor finished = by_beam(args[Finished], "finished", shape, device);
    TORCH_CHECK(!finished.defined() || finished.scalar_type() == at::kBool, "tensor finished must have dtype bool, got ",
                finished.scalar_type());
    const Tensor lengths = by_beam(args[Lengths], "lengths", shape, device);
    if (lengths.defined()) a.lengths_i64 = is_index(lengths, "lengths");
    a.length_penalty = number(args[LengthPenalty]);
    TORCH_CHECK_VALUE(a.length_penalty == 0.0 || lengths.defined(), "a length_penalty needs lengths");
    TORCH_CHECK_VALUE(a.length_penalty >= -8.0 && a.length_penalty <= 8.0, "length_penalty must be -8 to 8, got ",
                      a.length_penalty);
    a.pad = whole(args[Pad], "pad");
    a.searches = searches;
    a.beams = beams;
    a.vocab = vocab;
    a.n = count;
    a.logits = pointer(logits);
    a.search_stride = logits.stride(0);
    a.beam_stride = logits.stride(1);
    a.scores = static_cast<const float *>(pointer(scores));
    a.finished = static_cast<const uint8_t *>(pointer(finished));
    a.lengths = pointer(lengths);
    Tensor out_scores = fresh({searches, count}, at::kFloat, device);
    Tensor out_parents = fresh({searches, count}, at::kLong, device);
    Tensor out_tokens = fresh({searches, count}, at::kLong, device);
    a.out_scores = static_cast<float *>(out_scores.data_ptr());
    a.out_parents = static_cast<int64_t *>(out_parents.data_ptr());
    a.out_tokens = static_cast<int64_t *>(out_tokens.data_ptr());
    const uint64_t bytes = spiky_lm_beam_select_workspace(&a);
    Tensor workspace = fresh({(int64_t)bytes}, at::kByte, device);
    check(spiky_lm_beam_select(&a, workspace.data_ptr(), bytes, on.stream));
    return triple(out_scores, out_parents, out_tokens);
    END_HANDLE_TH_ERRORS
}

PyObject *reorder_states(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 3, "reorder_states takes 3 arguments");
    check_trace();
    enum { States, Parents, Out };
    bool one = false, one_out = false;
    const std::vector<PyObject *> given = each_of(args[States], one);
    std::vector<PyObject *> results;
    const bool to = args[Out] != Py_None;
    if (to) {
        results = each_of(args[Out], one_out);
        TORCH_CHECK_VALUE(results.size() == given.size() && one == one_out, "out must be as many tensors as states");
    }
    for (PyObject *o : given) check_tangent(o, "states");
    for (PyObject *o : results) check_tangent(o, "out");
    at::AutoGradMode off(false);
    Tensor parents = device_tensor(args[Parents], "parents");
    const bool i64 = is_index(parents, "parents");
    TORCH_CHECK_VALUE(parents.dim() == 2, "parents must be [B, n], got ", parents.sizes());
    const c10::Device device = parents.device();
    const int64_t searches = parents.size(0), count = parents.size(1);
    TORCH_CHECK_VALUE(count <= 4096, "parents must be of at most 4096 beams, got ", count);
    OnDevice on(device);
    parents = parents.contiguous();
    std::vector<Tensor> in(given.size()), out(given.size());
    std::vector<Side> from(given.size()), into(given.size());
    std::vector<spiky_lm_state> states(given.size());
    int64_t beams = 0;
    for (size_t i = 0; i < given.size(); i++) {
        // bits are moved: those that torch keeps beside the memory go into it first
        in[i] = device_tensor(given[i], "states", device);
        TORCH_CHECK(in[i].layout() == at::kStrided, "tensor states must be dense");
        if (in[i].is_conj()) in[i] = in[i].resolve_conj();
        TORCH_CHECK_VALUE(in[i].dim() >= 2 && in[i].size(0) == searches && (i == 0 || in[i].size(1) == beams),
                          "states must be [", searches, ", K, ...] of one K, got ", in[i].sizes());
        beams = in[i].size(1);
        const bool itself = to && results[i] == given[i];
        if (!side_of(in[i], from[i])) {
            TORCH_CHECK_VALUE(!itself, "a state that is reordered in place needs at most one dimension of runs that lie "
                                       "apart behind its beams");
            in[i] = in[i].contiguous();
            side_of(in[i], from[i]);
        }
        std::vector<int64_t> shape(in[i].sizes().begin(), in[i].sizes().end());
        shape[1] = count;
        if (to) {
            const Tensor &t = THPVariable_Check(results[i]) ? THPVariable_Unpack(results[i]) : Tensor();
            TORCH_CHECK(t.defined(), "tensor out must be a torch.Tensor");
            TORCH_CHECK(t.device() == device, "tensor out must be on ", device, ", got ", t.device());
            TORCH_CHECK_VALUE(!t.is_neg() && !t.is_conj(), "out must hold its values' signs");
            TORCH_CHECK_VALUE(t.sizes() == shape && t.scalar_type() == in[i].scalar_type(), "out must be ", shape, " of ",
                              in[i].scalar_type(), ", got ", t.sizes(), " of ", t.scalar_type());
            TORCH_CHECK_VALUE(!t.requires_grad(), "out must not require a gradient");
            out[i] = t;
            TORCH_CHECK_VALUE(side_of(t, into[i]), "out needs at most one dimension of runs that lie apart behind its beams");
        } else {
            out[i] = fresh(shape, in[i].scalar_type(), device);
            side_of(out[i], into[i]);
        }
        // runs of both sides alike: the longer ones are cut
        Side &a = from[i], &b = into[i];
        Side &longer = a.run_bytes > b.run_bytes ? a : b;
        const Side &shorter = a.run_bytes > b.run_bytes ? b : a;
        if (longer.run_bytes != shorter.run_bytes && in[i].numel() && out[i].numel()) {
            if (longer.runs == 1) {
                longer.run = (int64_t)shorter.run_bytes;
                longer.runs = shorter.runs;
                longer.run_bytes = shorter.run_bytes;
            } else {  // of which in place there are none
                in[i] = in[i].contiguous();
                side_of(in[i], a);
                a.run = (int64_t)b.run_bytes;
                a.runs = b.runs;
                a.run_bytes = b.run_bytes;
            }
        }
        const bool empty = in[i].numel() == 0 || out[i].numel() == 0;
        if (in[i].numel() == 0 && out[i].numel() > 0) out[i].zero_();  // of no beams, every parent is outside
        states[i] = {reinterpret_cast<const void *>(a.at), reinterpret_cast<void *>(b.at), empty ? 0 : a.runs,
                     a.run_bytes, a.search, a.beam, a.run, b.search, b.beam, b.run};
    }
    if (to && searches > 0 && count > 0) {
        Side by;
        by.at = reinterpret_cast<uintptr_t>(parents.data_ptr());
        by.run_bytes = parents.numel() * parents.element_size();
        const Bytes of_parents(by, 1, 1);
        std::vector<Bytes> source, target;
        std::vector<bool> in_place(given.size());
        for (size_t i = 0; i < given.size(); i++) {
            const Side &a = from[i], &b = into[i];
            source.emplace_back(a, searches, beams);
            target.emplace_back(b, searches, count);
            in_place[i] = a.at == b.at && a.search == b.search && a.beam == b.beam && a.run == b.run && a.runs == b.runs;
        }
        for (size_t i = 0; i < given.size(); i++) {
            if (out[i].numel() == 0) continue;
            const Bytes &b = target[i];
            TORCH_CHECK_VALUE(once_each(b), "the beams of out must not overlap");
            TORCH_CHECK_VALUE(b.end <= of_parents.at || of_parents.end <= b.at, "out must not overlap parents");
            TORCH_CHECK_VALUE(!in_place[i] || in[i].numel() == 0 || (count == beams && count <= 64),
                              "in place, parents must be [B, K] of at most 64 beams");
            for (size_t j = 0; j < given.size(); j++) {
                // a state in place of its result is looked at as that
                TORCH_CHECK_VALUE(in[j].numel() == 0 || in_place[j] || apart(source[j], b),
                                  "out must be its state, or share no memory with any");
                TORCH_CHECK_VALUE(j >= i || out[j].numel() == 0 || apart(target[j], b),
                                  "the tensors of out must share no memory");
            }
        }
    }
    check(spiky_lm_reorder(states.data(), states.size(), pointer(parents), i64, searches, beams, count, on.stream));
    if (to) {
        for (const Tensor &t : out)
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
        Py_INCREF(args[Out]);
        return args[Out];
    }
    if (one) return THPVariable_Wrap(out[0]);
    THPObjectPtr list(PyList_New((Py_ssize_t)out.size()));
    if (!list) throw python_error();
    for (size_t i = 0; i < out.size(); i++) PyList_SET_ITEM(list.get(), (Py_ssize_t)i, THPVariable_Wrap(out[i]));
    return list.release();
    END_HANDLE_TH_ERRORS
}

}  // namespace lm_torch
