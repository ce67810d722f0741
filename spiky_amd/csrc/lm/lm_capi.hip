// lm_capi.hip -- the C ABI of include/spiky_lm.h: host validation, and dispatch
// to the kernels on the caller's stream.  Nothing here allocates or synchronises.
#include <cmath>
#include <stdexcept>
#include <string>

#include "../../../include/spiky_lut.h"
#include "lm_kernels.h"

namespace {

thread_local std::string g_last_error;

struct ValueError : std::runtime_error {
    using std::runtime_error::runtime_error;
};

template <typename F>
int guarded(F &&f) {
    try {
        f();
        g_last_error.clear();
        return SPIKY_OK;
    } catch (const ValueError &e) {
        g_last_error = e.what();
        return SPIKY_VALUE_ERROR;
    } catch (const std::exception &e) {
        g_last_error = e.what();
        return SPIKY_RUNTIME_ERROR;
    } catch (...) {
        return SPIKY_RUNTIME_ERROR;
    }
}

void require(bool ok, const char *what) {
    if (!ok) throw ValueError(what);
}

void check_launch(hipError_t e, const char *what) {
    if (e != hipSuccess) throw std::runtime_error(std::string(what) + ": " + hipGetErrorString(e));
}

bool is_type(int t) { return t == SPIKY_F32 || t == SPIKY_BF16 || t == SPIKY_F16; }

spiky::lm::DropArgs drop_args(double p, uint64_t seed, uint64_t offset, const int64_t *rng) {
    require(p >= 0.0 && p <= 1.0, "dropout probability must be between 0 and 1");
    spiky::lm::DropArgs d;
    const double t = std::floor(p * 4294967296.0 + 0.5);
    d.threshold = t >= 4294967296.0 ? 0xffffffffu : (uint32_t)t;
    d.scale = t >= 4294967296.0 ? 0.f : (float)(1.0 / (1.0 - p));
    d.seed = seed;
    d.offset = offset;
    d.rng = rng;
    return d;
}

spiky::lm::DropArgs check(const spiky_lm_residual_args *a) {
    require(a != nullptr, "null pointer");
    require(is_type(a->res_dtype) && is_type(a->act_dtype), "unknown element type");
    require(a->res_dtype == a->act_dtype || a->res_dtype == SPIKY_F32,
            "the residual must be fp32 or have the branch's type");
    require(a->rows < 0x100000000ull && a->cols <= 0x4000000ull, "too many rows or columns");
    require(a->post_norm >= SPIKY_NORM_NONE && a->post_norm <= SPIKY_NORM_LAYER &&
                a->pre_norm >= SPIKY_NORM_NONE && a->pre_norm <= SPIKY_NORM_LAYER,
            "unknown norm");
    if (a->gate)
        require(a->gate_rows > 0 && a->rows % a->gate_rows == 0, "gate_rows must divide the rows");
    if (a->rows == 0 || a->cols == 0) return drop_args(a->dropout_p, 0, 0, nullptr);  // null pointers say nothing then
    require(a->post_norm != SPIKY_NORM_NONE || (!a->post_weight && !a->post_bias),
            "parameters of a norm that is not applied");
    require(a->pre_norm != SPIKY_NORM_NONE || (!a->pre_weight && !a->pre_bias),
            "parameters of a norm that is not applied");
    require(a->branch || a->pre_norm != SPIKY_NORM_NONE, "neither a branch nor a norm");
    require(a->branch || (!a->gate && a->post_norm == SPIKY_NORM_NONE), "a gate or norm of no branch");
    require(a->residual, "null pointer");
    return drop_args(a->branch ? a->dropout_p : 0.0, a->seed, a->offset, a->rng);
}

hipStream_t as_stream(void *s) { return reinterpret_cast<hipStream_t>(s); }

}  // namespace

extern "C" {

const char *spiky_lm_last_error(void) { return g_last_error.c_str(); }

int spiky_lm_dropout(const void *x, int64_t x_stride, void *y, uint64_t rows, uint64_t cols, int dtype,
                     double p, uint64_t seed, uint64_t offset, const int64_t *rng, void *stream) {
    return guarded([&] {
        require(is_type(dtype), "unknown element type");
        require(rows < 0x100000000ull && cols <= 0x3fffffff0ull, "too many rows or columns");
        const spiky::lm::DropArgs d = drop_args(p, seed, offset, rng);
        if (rows == 0 || cols == 0) return;
        require(x && y, "null pointer");
        check_launch(spiky::lm::launch_dropout(x, x_stride, y, rows, cols, dtype, d, as_stream(stream)), "dropout");
    });
}

int spiky_lm_residual_norm(const spiky_lm_residual_args *args, void *out, void *normed, void *stream) {
    return guarded([&] {
        const spiky::lm::DropArgs d = check(args);
        if (args->rows == 0 || args->cols == 0) return;
        require((!args->branch || out) && (args->pre_norm == SPIKY_NORM_NONE || normed), "null pointer");
        check_launch(spiky::lm::launch_residual_norm(*args, d, out, normed, as_stream(stream)), "residual_norm");
    });
}

uint64_t spiky_lm_residual_norm_workspace(const spiky_lm_residual_args *args, const spiky_lm_residual_grads *grads) {
    uint64_t bytes = 0;
    guarded([&] {
        check(args);
        require(grads != nullptr, "null pointer");
        if (args->rows > 0 && args->cols > 0) bytes = spiky::lm::residual_norm_workspace(*args, *grads);
    });
    return bytes;
}

int spiky_lm_residual_norm_backward(const spiky_lm_residual_args *args, const spiky_lm_residual_grads *grads,
                                    void *stream) {
    return guarded([&] {
        const spiky::lm::DropArgs d = check(args);
        require(grads != nullptr, "null pointer");
        if (args->rows == 0 || args->cols == 0) return;
        require(!grads->d_normed || args->pre_norm != SPIKY_NORM_NONE, "a gradient of no output");
        require(args->branch || (!grads->d_branch && !grads->d_gate), "a gradient of no input");
        require((args->post_weight || !grads->d_post_weight) && (args->post_bias || !grads->d_post_bias) &&
                    (args->pre_weight || !grads->d_pre_weight) && (args->pre_bias || !grads->d_pre_bias) &&
                    (args->gate || !grads->d_gate),
                "a gradient of no input");
        require(args->stats != nullptr, "the backward pass needs the forward's stats");
        const uint64_t need = spiky::lm::residual_norm_workspace(*args, *grads);
        require(grads->workspace_bytes >= need && (grads->workspace || need == 0), "residual_norm workspace too small");
        check_launch(spiky::lm::launch_residual_norm_backward(*args, d, *grads, as_stream(stream)),
                     "residual_norm_backward");
    });
}

int spiky_lm_process_logits(const spiky_lm_logits_args *a, void *stream) {
    return guarded([&] {
        require(a != nullptr, "null pointer");
        require(is_type(a->dtype) && is_type(a->out_dtype), "unknown element type");
        require(a->out_dtype == a->dtype || a->out_dtype == SPIKY_F32,
                "the result must be fp32 or have the logits' type");
        require(!a->bias || is_type(a->bias_dtype), "unknown element type");
        require(a->vocab < 0x80000000ull, "too many entries");
        require(a->history < 0x40000000ull, "too long a history");
        require(!a->tokens || a->repetition_rows || a->repetition > 0.f, "repetition penalty must be positive");
        require(!a->bias_ids || a->bias_values, "bias ids without values");
        if (a->rows == 0 || a->vocab == 0) return;
        require(a->logits && a->out, "null pointer");
        check_launch(spiky::lm::launch_process_logits(*a, as_stream(stream)), "process_logits");
    });
}

}  // extern "C"
