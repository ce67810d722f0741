// lm_capi.hip -- the C ABI of include/spiky_lm.h and include/spiky_lm_tokens.h: host
// validation, and dispatch to the kernels on the caller's stream.  Nothing here allocates or synchronises.
#include <cmath>
#include <stdexcept>
#include <string>

#include "../../../include/spiky_lut.h"
#include "lm_kernels.h"
#include "lm_tokens.h"

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

void check(const spiky_lm_embed_args *a) {
    require(a != nullptr, "null pointer");
    require(is_type(a->weight_dtype) && is_type(a->out_dtype), "unknown element type");
    require(a->weight_dtype == a->out_dtype || a->weight_dtype == SPIKY_F32 || a->out_dtype == SPIKY_F32,
            "the table and the result must have one type, or one of them fp32");
    require(a->n < 0x80000000ull && a->vocab < 0x80000000ull && a->cols <= 0x800000ull,
            "too many tokens, rows or columns");
    require(std::isfinite((float)a->scale), "the scale must be finite in 32 bits");
}

void check(const spiky_lm_beams_args *a) {
    require(a != nullptr, "null pointer");
    require(is_type(a->dtype), "unknown element type");
    require(a->beams >= 1 && a->beams <= 64 && a->n >= 1 && a->n <= 64, "beams and n must be 1 to 64");
    require(a->vocab < 0x80000000ull && a->searches < 0x1000000ull / a->beams, "too many searches or entries");
    require(a->length_penalty >= -8.0 && a->length_penalty <= 8.0, "the length penalty must be -8 to 8");
}

void check(const spiky_lm_state &s) {
    require(s.run_bytes < (1ull << 35), "too long a run");
    require(s.runs == 0 || s.run_bytes == 0 || (s.in && s.out), "null pointer");
    require(s.runs == 0 || (s.run_bytes + 15) / 16 <= (1ull << 56) / s.runs, "too large a state");
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

int spiky_lm_embed(const spiky_lm_embed_args *a, void *out, void *stream) {
    return guarded([&] {
        check(a);
        if (a->n == 0 || a->cols == 0) return;
        require(a->tokens && (a->weight || a->vocab == 0) && out, "null pointer");
        check_launch(spiky::lm::launch_embed(*a, out, as_stream(stream)), "embed");
    });
}

uint64_t spiky_lm_embed_workspace(const spiky_lm_embed_args *a) {
    uint64_t bytes = 0;
    guarded([&] {
        check(a);
        if (a->vocab > 0 && a->cols > 0) bytes = spiky::lm::embed_workspace(*a);
    });
    return bytes;
}

int spiky_lm_embed_backward(const spiky_lm_embed_args *a, const void *d_out, int64_t d_out_stride, void *d_weight,
                            void *workspace, uint64_t workspace_bytes, void *stream) {
    return guarded([&] {
        check(a);
        if (a->vocab == 0 || a->cols == 0) return;
        require(d_weight && (a->n == 0 || (a->tokens && d_out)), "null pointer");
        require(workspace && workspace_bytes >= spiky::lm::embed_workspace(*a), "embed workspace too small");
        check_launch(spiky::lm::launch_embed_backward(*a, d_out, d_out_stride, d_weight, workspace, as_stream(stream)),
                     "embed_backward");
    });
}

uint64_t spiky_lm_beam_select_workspace(const spiky_lm_beams_args *a) {
    uint64_t bytes = 0;
    guarded([&] {
        check(a);
        bytes = spiky::lm::beam_select_workspace(*a);
    });
    return bytes;
}

int spiky_lm_beam_select(const spiky_lm_beams_args *a, void *workspace, uint64_t workspace_bytes, void *stream) {
    return guarded([&] {
        check(a);
        if (a->searches == 0) return;
        require(a->scores && a->out_scores && a->out_parents && a->out_tokens && (a->logits || a->vocab == 0),
                "null pointer");
        const uint64_t need = spiky::lm::beam_select_workspace(*a);
        require(workspace_bytes >= need && (workspace || need == 0), "beam_select workspace too small");
        check_launch(spiky::lm::launch_beam_select(*a, workspace, as_stream(stream)), "beam_select");
    });
}

int spiky_lm_reorder(const spiky_lm_state *states, uint64_t count, const void *parents, int parents_i64,
                     uint64_t searches, uint64_t beams, uint64_t n, void *stream) {
    return guarded([&] {
        require(states || count == 0, "null pointer");
        require(searches < 0x80000000ull && beams < 0x80000000ull && n <= 4096, "too many searches or beams");
        for (uint64_t i = 0; i < count; i++) {
            const spiky_lm_state &s = states[i];
            check(s);
            if (s.in != s.out || s.runs == 0) continue;
            require(n == beams && n <= 64, "in place, n must be the number of beams, at most 64");
            require((searches <= 1 || s.in_search == s.out_search) && (beams <= 1 || s.in_beam == s.out_beam) &&
                        (s.runs == 1 || s.in_run == s.out_run),
                    "in place, both strides must be the same");
        }
        if (searches == 0 || n == 0) return;
        require(parents != nullptr, "null pointer");
        check_launch(spiky::lm::launch_reorder(states, count, parents, parents_i64 != 0, searches, beams, n,
                                               as_stream(stream)),
                     "reorder");
    });
}

}  // extern "C"
