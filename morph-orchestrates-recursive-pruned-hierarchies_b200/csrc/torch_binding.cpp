// The dense site's operators on torch tensors: argument checks, allocations, the launch on the current
// stream of the tensors' device, and the autograd rules, in C++ above the C ABI.  A kernel of this site runs
// for a few microseconds on a small batch; the same steps in Python took 10 to 19 us a call and 115 us a
// training step of the layer norm.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>
#include <algorithm>
#include <atomic>
#include <optional>
#include <string>
#include <tuple>
#include <unordered_set>
#include <vector>
#include "mortar_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ---- launches counted per kernel family -------------------------------------------------------

enum Family { kLayerNorm, kLayerNormBackward, kDense, kDenseBackward, kQuantize, kDequantize, kLinearFp8, kFamilies };
const char *const kFamilyName[kFamilies] = {"layer_norm", "layer_norm_backward", "dense", "dense_backward",
                                            "quantize_fp8", "dequantize_fp8", "linear_fp8"};
std::atomic<long long> g_launches[kFamilies];

void count(Family f, long long n) { g_launches[f].fetch_add(n, std::memory_order_relaxed); }

// ---- checks and errors ------------------------------------------------------------------------

// Statuses as the ctypes binding turns them into exceptions: what is wrong with the arguments is a ValueError.
void check(int64_t status, const char *where) {
    if (status >= 0) return;
    std::string text = std::string(where) + ": " + mortar_status_string((int)status);
    if (status == MORTAR_ERR_CUDA) text += std::string(": ") + mortar_last_cuda_error();
    text += " (status " + std::to_string(status) + ")";
    TORCH_CHECK_VALUE(status < MORTAR_ERR_CAPACITY, text);
    TORCH_CHECK(false, text);
}

void need_cuda(const Tensor &t, const char *name) {
    TORCH_CHECK_NOT_IMPLEMENTED(t.is_cuda(), name, " is on ", t.device(),
                                ": the MORTAR operators are CUDA-only (sm_100a), no CPU path");
}
void same_device(const Tensor &t, const char *name, const Tensor &other) {
    TORCH_CHECK_VALUE(other.device() == t.device(), name, " is on ", other.device(), ", expected ", t.device());
}

int code_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return MORTAR_F32;
        case at::kBFloat16: return MORTAR_BF16;
        case at::kHalf: return MORTAR_F16;
        case at::kFloat8_e4m3fn: return MORTAR_E4M3;
        case at::kFloat8_e5m2: return MORTAR_E5M2;
        default: return -1;
    }
}
bool is_float(int code) { return code >= MORTAR_F32 && code <= MORTAR_F16; }
bool is_fp8(int code) { return code == MORTAR_E4M3 || code == MORTAR_E5M2; }

bool wants_grad(std::initializer_list<const Tensor *> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// No operator here has a forward-mode derivative.  A tangent is no gradient that is required (and stays on where none are
// recorded), so it is asked for by itself: without this the kernels would drop it in silence.
void refuse_tangents(const char *name, std::initializer_list<const Tensor *> ts) {
    for (const Tensor *t : ts)
        TORCH_CHECK_VALUE(!t->defined() || !t->unsafeGetTensorImpl()->_fw_grad(0, *t).defined(), name,
                          " has no forward-mode derivative: give it the primal of a dual tensor");
}

// The 8-bit operators record no gradient.
void refuse_gradients(const char *name, std::initializer_list<const Tensor *> ts) {
    TORCH_CHECK_VALUE(!wants_grad(ts), name, " is not differentiable: detach its inputs or call it under torch.no_grad()");
}

// ---- layouts ----------------------------------------------------------------------------------

// [..., cols] -> [rows, cols]
Tensor rows2d(const Tensor &t) { return t.dim() == 2 ? t : t.reshape({-1, t.size(-1)}); }

// The rows themselves when each is contiguous and none overlaps the next, else a copy (`aligned`: also when they do
// not start on 16 bytes).
Tensor rows_of(const Tensor &t, bool aligned) {
    const Tensor r = rows2d(t);
    const int64_t per16 = 16 / (int64_t)r.element_size();
    const bool ok = r.stride(1) == 1 && r.stride(0) >= r.size(1) && !r.is_neg() &&
                    (!aligned || (r.stride(0) % per16 == 0 && reinterpret_cast<uintptr_t>(r.const_data_ptr()) % 16 == 0));
    return ok ? r : r.clone(at::MemoryFormat::Contiguous);
}
// elements from row to row (a copy of one row may keep a stride that says nothing)
int64_t ld(const Tensor &rows) { return std::max(rows.stride(0), rows.size(1)); }

// memory holds the values themselves, one after the other
bool plain(const Tensor &t) { return t.is_contiguous() && !t.is_neg(); }

// Rows that the kernels may walk at `ld(t)` as they are: none lies over the next.
bool apart(const Tensor &t) { return t.size(0) < 2 || t.stride(0) >= t.size(1); }

Tensor like(const Tensor &t) { return t.is_contiguous() ? at::empty_like(t) : at::empty(t.sizes(), t.options()); }
Tensor floats(at::IntArrayRef shape, const Tensor &on) { return at::empty(shape, on.options().dtype(at::kFloat)); }
const void *in(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *out(const Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
float *out_f32(const Tensor &t) { return static_cast<float *>(out(t)); }
const float *in_f32(const Tensor &t) { return static_cast<const float *>(in(t)); }

// a gradient that no row contributes to
Tensor zeroed(const Tensor &t) { return t.defined() ? t.zero_() : t; }

struct Launch {                                       // the device of a tensor and its current stream
    c10::cuda::CUDAGuard guard;
    void *stream;
    explicit Launch(const Tensor &t)
        : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

Tensor or_none(const OptTensor &t) { return t.has_value() ? *t : Tensor(); }

void refuse_second(const char *name) {
    TORCH_CHECK(!at::GradMode::is_enabled(), name, " has no second derivative: call backward without create_graph");
}

// A leaf's gradient is accumulated on the stream that was current when the oldest living graph took the leaf up.
// A backward pass that is being captured cannot make the default stream wait for it: the capture fails inside the
// autograd engine, and the process ends with it.  So a forward call under capture refuses when a leaf above it is so
// held.  (The walk runs while a graph is captured, never in an eager step.)
void refuse_capture(const char *name, at::ArrayRef<const Tensor *> ts) {
    using torch::autograd::Node;
    const c10::cuda::CUDAGuard guard(ts.front()->device());
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
    std::vector<std::shared_ptr<Node>> todo;
    std::unordered_set<Node *> seen;
    const auto visit = [&](const std::shared_ptr<Node> &node) {
        if (node && seen.insert(node.get()).second) todo.push_back(node);
    };
    for (const Tensor *t : ts)
        if (t->defined() && t->requires_grad())
            visit(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
    while (!todo.empty()) {
        const std::shared_ptr<Node> node = todo.back();
        todo.pop_back();
        for (const auto &edge : node->next_edges()) visit(edge.function);
        if (node->num_outputs() != 0) continue;          // not a leaf's accumulator
        const auto s = node->stream();
        TORCH_CHECK(!s.has_value() || c10::cuda::CUDAStream(*s).stream() != nullptr, name,
                    ": a tensor whose gradient a graph from the default stream still holds cannot be part of a captured "
                    "training step: drop that graph's outputs first, or detach them");
    }
}

// ---- layer norm -------------------------------------------------------------------------------

Tensor as_f32(const Tensor &t) {
    if (!t.defined() || (t.scalar_type() == at::kFloat && t.is_contiguous() && !t.is_neg())) return t;
    return t.detach().to(at::kFloat).contiguous().resolve_neg();
}

void check_columns(const Tensor &x, const char *name, const Tensor &t) {
    if (!t.defined()) return;
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == x.size(-1) && is_float(code_of(t.scalar_type())), name,
                      " must be a float tensor [", x.size(-1), "], got ", t.scalar_type(), " ", t.sizes());
    same_device(x, name, t);
}

std::tuple<Tensor, Tensor> layer_norm_forward(const Tensor &x, const Tensor &weight, const Tensor &bias, double eps,
                                              bool want_stats) {
    need_cuda(x, "x");
    refuse_tangents("layer_norm", {&x, &weight, &bias});
    const int code = code_of(x.scalar_type());
    TORCH_CHECK_VALUE(is_float(code) && x.dim() >= 1, "x must be a float32, bfloat16 or float16 tensor [..., cols], got ",
                      x.scalar_type());
    const int64_t cols = x.size(-1);
    TORCH_CHECK_VALUE(cols >= 1, "the last dimension is empty: a mean of nothing is not defined");
    TORCH_CHECK_VALUE(cols <= INT32_MAX, "rows of ", cols, " columns are not supported");
    check_columns(x, "weight", weight);
    check_columns(x, "bias", bias);
    const Launch on(x);
    const Tensor y = like(x), r = rows_of(x, false);
    const int64_t rows = r.size(0);
    Tensor stats;
    if (want_stats) stats = floats({2, rows}, x);
    if (rows == 0) return {y, stats};
    const Tensor w = as_f32(weight), b = as_f32(bias);
    check(mortar_layer_norm(in(r), code, ld(r), rows, (int32_t)cols, in_f32(w), in_f32(b), (float)eps, out(y), cols,
                            out_f32(stats), on.stream), "mortar_layer_norm");
    count(kLayerNorm, 1);
    return {y, stats};
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward(const Tensor &dy, const Tensor &x, const Tensor &weight,
                                                       const Tensor &stats, bool want_dx, bool want_dweight,
                                                       bool want_dbias) {
    need_cuda(x, "x");
    refuse_tangents("layer_norm_backward", {&dy, &x, &weight});
    const int code = code_of(x.scalar_type());
    TORCH_CHECK_VALUE(is_float(code) && x.dim() >= 1 && x.size(-1) >= 1 && dy.sizes() == x.sizes(), "dy has shape ",
                      dy.sizes(), ", x ", x.sizes(), " (", x.scalar_type(), ")");
    same_device(x, "dy", dy);
    same_device(x, "stats", stats);
    check_columns(x, "weight", weight);
    const int64_t cols = x.size(-1), rows = x.numel() / cols;
    TORCH_CHECK_VALUE(stats.scalar_type() == at::kFloat && stats.dim() == 2 && stats.size(0) == 2 && stats.size(1) == rows &&
                          plain(stats), "stats must be contiguous float32 [2, ", rows, "]");
    const Launch on(x);
    Tensor dx, dw, db, scratch;
    if (want_dx) dx = like(x);
    if (want_dweight) dw = floats({cols}, x);
    if (want_dbias) db = floats({cols}, x);
    if (rows == 0) return {dx, zeroed(dw), zeroed(db)};
    if (!want_dx && !want_dweight && !want_dbias) return {dx, dw, db};
    const Tensor d = rows_of(dy.scalar_type() == x.scalar_type() ? dy : dy.to(x.scalar_type()), false);
    const Tensor r = rows_of(x, false), w = as_f32(weight);
    int64_t n = 0;
    if (want_dweight || want_dbias) {
        n = mortar_layer_norm_scratch_floats(rows, (int32_t)cols);
        check(n, "mortar_layer_norm_scratch_floats");
        scratch = floats({n}, x);
    }
    check(mortar_layer_norm_backward(in(d), ld(d), in(r), ld(r), code, rows, (int32_t)cols, in_f32(w), in_f32(stats),
                                     out(dx), cols, out_f32(dw), out_f32(db), out_f32(scratch), n, on.stream),
          "mortar_layer_norm_backward");
    count(kLayerNormBackward, n ? 2 : 1);
    return {dx, dw, db};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const OptTensor &weight, const OptTensor &bias, double eps) {
        auto [y, stats] = layer_norm_forward(x, or_none(weight), or_none(bias), eps, true);
        ctx->save_for_backward({x, or_none(weight), stats});
        ctx->saved_data["bias"] = bias.has_value() ? (int64_t)bias->scalar_type() : (int64_t)-1;
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        refuse_second("layer_norm");
        const auto saved = ctx->get_saved_variables();
        const int64_t bias = ctx->saved_data["bias"].toInt();
        size_t edge = 0;                                 // edges exist for the tensors that were given
        const bool need_x = ctx->needs_input_grad(edge++);
        const bool need_w = saved[1].defined() && ctx->needs_input_grad(edge++);
        const bool need_b = bias >= 0 && ctx->needs_input_grad(edge++);
        auto [dx, dw, db] = layer_norm_backward(grads[0], saved[0], saved[1], saved[2], need_x, need_w, need_b);
        if (dw.defined() && saved[1].scalar_type() != at::kFloat) dw = dw.to(saved[1].scalar_type());
        if (db.defined() && (at::ScalarType)bias != at::kFloat) db = db.to((at::ScalarType)bias);
        return {dx, dw, db, Tensor()};
    }
};

Tensor layer_norm(const Tensor &x, const OptTensor &weight, const OptTensor &bias, double eps) {
    const Tensor w = or_none(weight), b = or_none(bias);
    if (wants_grad({&x, &w, &b})) {
        need_cuda(x, "x");
        refuse_tangents("layer_norm", {&x, &w, &b});        // inside `apply` forward mode is off
        refuse_capture("layer_norm", {&x, &w, &b});
        return LayerNorm::apply(x, weight, bias, eps);
    }
    return std::get<0>(layer_norm_forward(x, w, b, eps, false));
}

// ---- the dense block --------------------------------------------------------------------------

struct MlpShape { int64_t d_model, d_ff; int code; };

MlpShape check_mlp(const Tensor &x, const Tensor &gate_up, const Tensor &down) {
    need_cuda(x, "x");
    const auto dt = x.scalar_type();
    TORCH_CHECK_VALUE(dt == at::kBFloat16 || dt == at::kHalf, "mlp_dense takes bfloat16 or float16 activations, got ", dt);
    TORCH_CHECK_VALUE(x.dim() >= 1 && gate_up.dim() == 2 && down.dim() == 2,
                      "x [..., d_model], gate_up [2 d_ff, d_model] and down [d_model, d_ff] expected");
    const int64_t d_model = down.size(0), d_ff = down.size(1);
    TORCH_CHECK_VALUE(gate_up.size(0) == 2 * d_ff && gate_up.size(1) == d_model && x.size(-1) == d_model, "x ", x.sizes(),
                      ", gate_up ", gate_up.sizes(), " and down ", down.sizes(),
                      " do not fit: x [..., d_model], gate_up [2 d_ff, d_model] and down [d_model, d_ff] expected");
    TORCH_CHECK_VALUE(d_model >= 1 && d_ff >= 1 && d_model % 16 == 0 && d_ff % 16 == 0,
                      "d_model and d_ff must be positive multiples of 16, got ", d_model, " and ", d_ff);
    TORCH_CHECK_VALUE(d_model <= (1 << 29) && d_ff <= (1 << 29), "d_model ", d_model, " or d_ff ", d_ff, " is too large");
    TORCH_CHECK_VALUE(gate_up.scalar_type() == dt && down.scalar_type() == dt, "gate_up is ", gate_up.scalar_type(),
                      ", down ", down.scalar_type(), " and x ", dt, ": one type for all");
    same_device(x, "gate_up", gate_up);
    same_device(x, "down", down);
    return {d_model, d_ff, code_of(dt)};
}

std::tuple<Tensor, Tensor, Tensor> mlp_dense_forward(const Tensor &x, const Tensor &gate_up, const Tensor &down,
                                                     bool want_saved) {
    const MlpShape s = check_mlp(x, gate_up, down);
    refuse_tangents("mlp_dense", {&x, &gate_up, &down});
    const Launch on(x);
    const Tensor r = rows_of(x, true), gu = rows_of(gate_up, true), dn = rows_of(down, true);
    const int64_t rows = r.size(0);
    const Tensor y = like(x), hidden = at::empty({rows, s.d_ff}, x.options());
    Tensor sums, scratch;
    if (want_saved) sums = floats({rows, 2 * s.d_ff}, x);
    if (rows == 0) return {y, hidden, sums};
    const int64_t n = mortar_mlp_dense_scratch_floats(rows, (int32_t)s.d_model, (int32_t)s.d_ff, want_saved);
    check(n, "mortar_mlp_dense_scratch_floats");
    if (n) scratch = floats({n}, x);
    check(mortar_mlp_dense(in(r), ld(r), s.code, rows, in(gu), ld(gu), in(dn), ld(dn), (int32_t)s.d_model, (int32_t)s.d_ff,
                           out(hidden), out_f32(sums), out(y), s.d_model, out_f32(scratch), n, on.stream),
          "mortar_mlp_dense");
    count(kDense, n ? 3 : 2);
    return {y, hidden, sums};
}

std::tuple<Tensor, Tensor, Tensor> mlp_dense_backward(const Tensor &dy, const Tensor &x, const Tensor &gate_up,
                                                      const Tensor &down, const Tensor &hidden, const Tensor &sums,
                                                      bool want_dx, bool want_dgate_up, bool want_ddown) {
    const MlpShape s = check_mlp(x, gate_up, down);
    refuse_tangents("mlp_dense_backward", {&dy, &x, &gate_up, &down});
    TORCH_CHECK_VALUE(dy.sizes() == x.sizes(), "dy has shape ", dy.sizes(), ", x ", x.sizes());
    same_device(x, "dy", dy);
    same_device(x, "hidden", hidden);
    same_device(x, "sums", sums);
    const auto dt = x.scalar_type();
    const int64_t rows = x.numel() / s.d_model;
    TORCH_CHECK_VALUE(hidden.dim() == 2 && hidden.size(0) == rows && hidden.size(1) == s.d_ff && hidden.scalar_type() == dt &&
                          plain(hidden), "hidden must be contiguous ", dt, " [", rows, ", ", s.d_ff, "]");
    TORCH_CHECK_VALUE(sums.dim() == 2 && sums.size(0) == rows && sums.size(1) == 2 * s.d_ff && sums.scalar_type() == at::kFloat &&
                          plain(sums), "sums must be contiguous float32 [", rows, ", ", 2 * s.d_ff, "]");
    const Launch on(x);
    Tensor dx, dgu, ddn, scratch;
    if (want_dx) dx = like(x);
    if (want_dgate_up) dgu = at::empty({2 * s.d_ff, s.d_model}, x.options());
    if (want_ddown) ddn = at::empty({s.d_model, s.d_ff}, x.options());
    if (rows == 0) return {dx, zeroed(dgu), zeroed(ddn)};
    if (!want_dx && !want_dgate_up && !want_ddown) return {dx, dgu, ddn};
    const Tensor d = rows_of(dy.scalar_type() == dt ? dy : dy.to(dt), true), r = rows_of(x, true);
    const Tensor gu = rows_of(gate_up, true), dn = rows_of(down, true);
    const Tensor dsums = at::empty({rows, 2 * s.d_ff}, x.options());
    const int64_t n = mortar_mlp_dense_backward_scratch_floats(rows, (int32_t)s.d_model, (int32_t)s.d_ff, want_dx,
                                                               want_dgate_up, want_ddown);
    check(n, "mortar_mlp_dense_backward_scratch_floats");
    if (n) scratch = floats({n}, x);
    check(mortar_mlp_dense_backward(in(d), ld(d), in(r), ld(r), s.code, rows, in(gu), ld(gu), in(dn), ld(dn),
                                    (int32_t)s.d_model, (int32_t)s.d_ff, in(hidden), in_f32(sums), out(dsums), out(dx),
                                    out(dgu), out(ddn), out_f32(scratch), n, on.stream), "mortar_mlp_dense_backward");
    count(kDenseBackward, (want_dx || want_dgate_up ? 1 : 0) + (n ? 2 : 1));
    return {dx, dgu, ddn};
}

struct MlpDense : torch::autograd::Function<MlpDense> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &gate_up, const Tensor &down) {
        auto [y, hidden, sums] = mlp_dense_forward(x, gate_up, down, true);
        ctx->save_for_backward({x, gate_up, down, hidden, sums});
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        refuse_second("mlp_dense");
        const auto s = ctx->get_saved_variables();
        auto [dx, dgu, ddn] = mlp_dense_backward(grads[0], s[0], s[1], s[2], s[3], s[4], ctx->needs_input_grad(0),
                                                 ctx->needs_input_grad(1), ctx->needs_input_grad(2));
        return {dx, dgu, ddn};
    }
};

Tensor mlp_dense(const Tensor &x, const Tensor &gate_up, const Tensor &down) {
    if (wants_grad({&x, &gate_up, &down})) {
        need_cuda(x, "x");
        refuse_tangents("mlp_dense", {&x, &gate_up, &down});
        refuse_capture("mlp_dense", {&x, &gate_up, &down});
        return MlpDense::apply(x, gate_up, down);
    }
    return std::get<0>(mlp_dense_forward(x, gate_up, down, false));
}

// ---- 8-bit floating point ---------------------------------------------------------------------

std::tuple<Tensor, Tensor> quantize_fp8(const Tensor &x, int64_t block_rows, at::ScalarType dtype) {
    need_cuda(x, "x");
    refuse_tangents("quantize_fp8", {&x});
    refuse_gradients("quantize_fp8", {&x});
    const int code = code_of(x.scalar_type()), q_code = code_of(dtype);
    TORCH_CHECK_VALUE(x.dim() == 2 && is_float(code), "quantize_fp8 takes a 2-D float32, bfloat16 or float16 tensor, got ",
                      x.scalar_type(), " ", x.sizes());
    TORCH_CHECK_VALUE(is_fp8(q_code), "dtype must be float8_e4m3fn or float8_e5m2, got ", dtype);
    TORCH_CHECK_VALUE(block_rows == 1 || block_rows == 128, "block_rows must be 1 or 128, got ", block_rows);
    const int64_t rows = x.size(0), cols = x.size(1);
    TORCH_CHECK_VALUE(cols >= 1 && cols % 16 == 0 && cols <= (1 << 30), "cols must be a positive multiple of 16 up to 2^30, got ", cols);
    const Launch on(x);
    const Tensor r = rows_of(x, true), q = at::empty({rows, cols}, x.options().dtype(dtype));
    const Tensor scale = floats({(rows + block_rows - 1) / block_rows, (cols + 127) / 128}, x);
    if (rows == 0) return {q, scale};
    check(mortar_quantize_fp8(in(r), code, ld(r), rows, (int32_t)cols, (int32_t)block_rows, out(q), q_code, cols,
                              out_f32(scale), on.stream), "mortar_quantize_fp8");
    count(kQuantize, 1);
    return {q, scale};
}

Tensor dequantize_fp8(const Tensor &q, const Tensor &scale, at::ScalarType out_dtype) {
    need_cuda(q, "q");
    refuse_tangents("dequantize_fp8", {&q, &scale});
    refuse_gradients("dequantize_fp8", {&q, &scale});
    const int q_code = code_of(q.scalar_type()), code = code_of(out_dtype);
    TORCH_CHECK_VALUE(q.dim() == 2 && is_fp8(q_code), "q must be a 2-D float8_e4m3fn or float8_e5m2 tensor, got ",
                      q.scalar_type(), " ", q.sizes());
    TORCH_CHECK_VALUE(is_float(code), "unsupported out_dtype ", out_dtype);
    const int64_t rows = q.size(0), cols = q.size(1), nb = (cols + 127) / 128, rb = (rows + 127) / 128;
    TORCH_CHECK_VALUE(cols >= 1 && cols % 16 == 0 && cols <= (1 << 30), "cols must be a positive multiple of 16 up to 2^30, got ", cols);
    TORCH_CHECK_VALUE(scale.scalar_type() == at::kFloat && scale.dim() == 2 && scale.size(1) == nb &&
                          (scale.size(0) == rows || scale.size(0) == rb), "scale must be float32 [", rows, ", ", nb, "] or [",
                      rb, ", ", nb, "], got ", scale.scalar_type(), " ", scale.sizes());
    same_device(q, "scale", scale);
    const Launch on(q);
    const Tensor y = at::empty({rows, cols}, q.options().dtype(out_dtype));
    if (rows == 0) return y;
    const Tensor r = rows_of(q, true), s = scale.contiguous().resolve_neg();
    check(mortar_dequantize_fp8(in(r), q_code, ld(r), in_f32(s), rows, (int32_t)cols, scale.size(0) == rows ? 1 : 128, out(y),
                                code, cols, on.stream), "mortar_dequantize_fp8");
    count(kDequantize, 1);
    return y;
}

Tensor linear_fp8(const Tensor &x, const OptTensor &x_scale, const Tensor &data, const Tensor &scale, bool swiglu,
                  const std::optional<at::ScalarType> &out_dtype) {
    need_cuda(x, "x");
    const int code = code_of(x.scalar_type());
    TORCH_CHECK_VALUE(code >= 0 && x.dim() >= 1, "x must be a float or float8 tensor [..., in], got ", x.scalar_type());
    TORCH_CHECK_VALUE(x_scale.has_value() == is_fp8(code), "x_scale goes with an 8-bit x, and only with one");
    TORCH_CHECK_VALUE(data.dim() == 2 && is_fp8(code_of(data.scalar_type())), "w.data must be a float8 matrix, got ",
                      data.scalar_type(), " ", data.sizes());
    const int64_t n = data.size(0), k = data.size(1), nb = (k + 127) / 128;
    TORCH_CHECK_VALUE(data.stride(1) == 1 && scale.scalar_type() == at::kFloat && scale.dim() == 2 &&
                          scale.size(0) == (n + 127) / 128 && scale.size(1) == nb && scale.stride(1) == 1,
                      "w.scale must be float32 [", (n + 127) / 128, ", ", nb, "], got ", scale.scalar_type(), " ", scale.sizes());
    TORCH_CHECK_VALUE(!data.is_neg() && !scale.is_neg(), "w.data or w.scale is a view of negative values: pass a copy");
    TORCH_CHECK_VALUE(apart(data) && apart(scale), "the rows of w.data or w.scale overlap (strides ", data.strides(), " and ",
                      scale.strides(), "): pass a contiguous copy");
    TORCH_CHECK_VALUE(x.size(-1) == k, "x has last dim ", x.size(-1), ", expected ", k);
    TORCH_CHECK_VALUE(n <= INT32_MAX && k <= INT32_MAX, "a matrix [", n, ", ", k, "] is too large");
    const Tensor given = or_none(x_scale);
    refuse_tangents("linear_fp8", {&x, &given, &data, &scale});
    refuse_gradients("linear_fp8", {&x, &given, &data, &scale});
    TORCH_CHECK_VALUE(!swiglu || n % 256 == 0, "swiglu needs out_features to be a multiple of 256, got ", n);
    const at::ScalarType y_type = out_dtype.value_or(is_float(code) ? x.scalar_type() : at::kBFloat16);
    const int y_code = code_of(y_type);
    TORCH_CHECK_VALUE(is_float(y_code), "unsupported out_dtype ", y_type);
    same_device(x, "w", data);
    same_device(x, "w.scale", scale);
    if (given.defined()) {
        same_device(x, "x_scale", given);
        bool fits = given.scalar_type() == at::kFloat && given.dim() == x.dim() && given.size(-1) == nb;
        for (int64_t i = 0; fits && i + 1 < x.dim(); ++i) fits = given.size(i) == x.size(i);
        TORCH_CHECK_VALUE(fits, "x_scale must be float32 with the leading dimensions of x and ", nb, " blocks, got ",
                          given.scalar_type(), " ", given.sizes());
    }
    const Launch on(x);
    const int64_t n_out = swiglu ? n / 2 : n;
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = n_out;
    const Tensor y = at::empty(shape, x.options().dtype(y_type));
    Tensor r = rows2d(x), s;
    const int64_t rows = r.size(0);
    if (rows == 0) return y;
    if (given.defined()) {
        r = rows_of(x, true);
        s = rows_of(given, false);
        if (ld(s) > UINT32_MAX / rows) s = s.clone(at::MemoryFormat::Contiguous);     // the kernels keep 32-bit positions of scales
    } else {
        std::tie(r, s) = quantize_fp8(r, 1, at::kFloat8_e4m3fn);
    }
    const int32_t flags = swiglu ? MORTAR_FLAG_SWIGLU : 0;
    const int64_t scratch_floats = mortar_linear_fp8_scratch_floats(rows, (int32_t)n, (int32_t)k, flags);
    check(scratch_floats, "mortar_linear_fp8_scratch_floats");
    Tensor scratch;
    if (scratch_floats) scratch = floats({scratch_floats}, x);
    check(mortar_linear_fp8_cut(in(r), code_of(r.scalar_type()), ld(r), in_f32(s), ld(s), rows, in(data),
                                code_of(data.scalar_type()), ld(data), in_f32(scale), ld(scale), (int32_t)n, (int32_t)k, flags,
                                out(y), y_code, n_out, out_f32(scratch), scratch_floats, on.stream), "mortar_linear_fp8");
    count(kLinearFp8, scratch_floats ? 2 : 1);
    return y;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    namespace py = pybind11;
    // no call touches a Python object: other threads run meanwhile, as with torch's own operators
    const py::call_guard<py::gil_scoped_release> no_gil;
    m.def("refuse_capture", [](const std::string &name, const std::vector<OptTensor> &ts) {
        std::vector<Tensor> held;
        std::vector<const Tensor *> at;
        for (const OptTensor &t : ts) held.push_back(or_none(t));
        for (const Tensor &t : held) at.push_back(&t);
        refuse_capture(name.c_str(), at);
    }, no_gil);
    m.def("layer_norm", &layer_norm, no_gil);
    m.def("layer_norm_forward", [](const Tensor &x, const OptTensor &w, const OptTensor &b, double eps, bool stats) {
        return layer_norm_forward(x, or_none(w), or_none(b), eps, stats);
    }, no_gil);
    m.def("layer_norm_backward", [](const Tensor &dy, const Tensor &x, const OptTensor &w, const Tensor &stats, bool dx,
                                    bool dw, bool db) { return layer_norm_backward(dy, x, or_none(w), stats, dx, dw, db); },
          no_gil);
    m.def("mlp_dense", &mlp_dense, no_gil);
    m.def("mlp_dense_forward", &mlp_dense_forward, no_gil);
    m.def("mlp_dense_backward", &mlp_dense_backward, no_gil);
    m.def("quantize_fp8", &quantize_fp8, no_gil);
    m.def("dequantize_fp8", &dequantize_fp8, no_gil);
    m.def("linear_fp8", &linear_fp8, no_gil);
    m.def("kernel_counts", [] {
        py::dict d;
        for (int i = 0; i < kFamilies; ++i)
            if (const long long n = g_launches[i].load()) d[kFamilyName[i]] = n;
        return d;
    });
}
