// The operators around a block as PyTorch functions with C++ autograd nodes, on top of the C ABI (include/loopback_b200.h).
//
// A decode step and the backward of a small batch are bound by what the host does per call: with Python autograd nodes and
// ctypes the norm's forward and backward took 108 us of host time around 66 us of kernels, and a decode step's norm 12 us around
// 2. The checks, the allocations and the nodes are here instead; loopback_b200/block.py gives them their names and documents
// them. The entry points are the ones ctypes resolved (bind), so there is one copy of the library whichever file it came from.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/loopback_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

#define LB_ENTRIES(X) \
    X(lb_last_error_string) X(lb_block_scratch_bytes) X(lb_norm_fwd) X(lb_norm_bwd) X(lb_residual_fwd) X(lb_residual_bwd) \
    X(lb_dropout) X(lb_ffn_workspace_bytes) X(lb_ffn_kept_bytes) X(lb_ffn_fwd) X(lb_ffn_bwd)

struct Entries {
#define LB_FIELD(name) decltype(&::name) name = nullptr;
    LB_ENTRIES(LB_FIELD)
#undef LB_FIELD
} lb;

void bind(const std::map<std::string, uintptr_t> &addresses) {
#define LB_BIND(name) lb.name = reinterpret_cast<decltype(&::name)>(addresses.at(#name));
    LB_ENTRIES(LB_BIND)
#undef LB_BIND
}

void check(int rc, const char *what) {
    TORCH_CHECK(rc == 0, "loopback_b200 ", what, " failed (status ", rc, "): ", lb.lb_last_error_string());
}

// the tensors' device made current, and its current stream
struct On {
    c10::cuda::CUDAGuard guard;
    void *stream;
    explicit On(const Tensor &t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
template <typename T> T *ptr_as(const Tensor &t) { return static_cast<T *>(ptr(t)); }

int code(const Tensor &t) {
    if (t.scalar_type() == at::kBFloat16) return LB_DTYPE_BF16;
    TORCH_CHECK(t.scalar_type() == at::kFloat, "loopback_b200 stores activations as bfloat16 or float32, got ", t.scalar_type());
    return LB_DTYPE_F32;
}

void require_rows(const Tensor &x, const char *what) {
    TORCH_CHECK(x.is_cuda(), "loopback_b200.", what, ": tensors must live on a CUDA device (there is no CPU path)");
    TORCH_CHECK(x.dim() > 0 && x.size(-1) > 0, "loopback_b200.", what, ": rows need a last dimension of at least one column, got shape ",
                x.sizes());
}

void same_device(const Tensor &x, const Tensor &t, const char *what) {
    TORCH_CHECK(!t.defined() || t.device() == x.device(), "loopback_b200.", what, ": a tensor is on ", t.device(), ", the rows are on ",
                x.device());
}

bool wants_grad(std::initializer_list<Tensor> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor &t : ts)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}

// contiguous and on a 16-byte boundary (a view may begin anywhere), a copy where it is not
Tensor dense(const Tensor &t) {
    Tensor c = t.contiguous();
    return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15) ? c.clone() : c;
}

Tensor bytes(size_t n, const Tensor &like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }
Tensor floats(int64_t n, const Tensor &like) { return at::empty({n}, like.options().dtype(at::kFloat)); }

// per-channel parameters in one storage type the kernels take: the rows' or, where they are fp32 or differ, fp32
void channel_params(const Tensor &x, std::initializer_list<Tensor *> ps, const char *what) {
    const int64_t d = x.size(-1);
    bool cast = false, seen = false;
    at::ScalarType kind = at::kFloat;
    for (const Tensor *p : ps) {
        if (!p->defined()) continue;
        same_device(x, *p, what);
        TORCH_CHECK(p->dim() == 1 && p->size(0) == d, "loopback_b200.", what, ": a per-channel parameter has shape ", p->sizes(),
                    ", rows have ", d, " columns");
        const at::ScalarType k = p->scalar_type();
        cast = cast || (seen && k != kind) || (k != x.scalar_type() && k != at::kFloat);
        kind = k;
        seen = true;
    }
    for (Tensor *p : ps)
        if (p->defined()) *p = dense(cast ? p->to(at::kFloat) : *p);
}

// The engine hands a gradient over on the stream of the node that takes it. While a backward is captured that must not be the
// default stream, which cannot be part of a capture: a leaf's node was made there where an eager graph of the same leaf is still
// alive. The engine's own error would end the process; this one is raised before it, and the capture ends in order.
void check_capture(const char *what) {
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    for (size_t i = 0; i < node->num_outputs(); ++i) {
        if (!node->task_should_compute_output(i)) continue;
        const auto s = node->next_edge(i).function->stream();
        TORCH_CHECK(!s || s->device_type() != c10::DeviceType::CUDA || c10::cuda::CUDAStream(*s).stream() != nullptr, "loopback_b200.", what,
                    ": this backward is captured into a CUDA graph, but an input's gradient belongs to the default stream: an eager "
                    "autograd graph of the same tensor is alive. Release its results before the capture, or record it on another stream");
    }
}

// Under create_graph the results of a backward would be taken for constants: they raise where somebody differentiates them.
variable_list once(variable_list grads, const char *what) {
    if (!at::GradMode::is_enabled()) return grads;
    for (Tensor &g : grads) {
        if (!g.defined()) continue;
        auto node = std::make_shared<torch::autograd::DelayedError>(std::string("loopback_b200.") + what + " is differentiable once", 1);
        g = node->apply({g.detach().requires_grad_()})[0];
    }
    return grads;
}

// ---------------------------------------------------------------------------------------------------------
// the norm before a block
// ---------------------------------------------------------------------------------------------------------
Tensor norm_forward(const Tensor &x, const Tensor &w, double eps, float *r) {
    const int64_t d = x.size(-1);
    Tensor u = at::empty_like(x);
    On on(x);
    check(lb.lb_norm_fwd(ptr(x), ptr(w), ptr(u), r, x.numel() / d, (int)d, (float)eps, code(x), code(w), on.stream), "block norm");
    return u;
}

struct BlockNorm : torch::autograd::Function<BlockNorm> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, double eps) {
        Tensor r = floats(x.numel() / x.size(-1), x);
        Tensor u = norm_forward(x, w, eps, ptr_as<float>(r));
        ctx->save_for_backward({x, w, r});
        return u;
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        check_capture("block_norm");
        const variable_list s = ctx->get_saved_variables();
        const Tensor &x = s[0], &w = s[1], &r = s[2];
        const int64_t d = x.size(-1);
        const Tensor du = dense(g[0]);
        Tensor dx, dw, scratch;
        if (ctx->needs_input_grad(0)) dx = at::empty_like(x);
        if (ctx->needs_input_grad(1)) {
            dw = at::empty_like(w);
            scratch = bytes(lb.lb_block_scratch_bytes((int)d), x);
        }
        On on(x);
        check(lb.lb_norm_bwd(ptr(x), ptr(w), ptr_as<float>(r), ptr(du), ptr(dx), ptr(dw), ptr(scratch), x.numel() / d, (int)d, code(x),
                             code(w), on.stream), "block norm backward");
        return once({dx, dw, Tensor()}, "block_norm");
    }
};

Tensor block_norm(const Tensor &x, Tensor w, double eps) {
    require_rows(x, "block_norm");
    channel_params(x, {&w}, "block_norm");
    const Tensor xc = dense(x);
    return wants_grad({xc, w}) ? BlockNorm::apply(xc, w, eps) : norm_forward(xc, w, eps, nullptr);
}

// ---------------------------------------------------------------------------------------------------------
// dropout
// ---------------------------------------------------------------------------------------------------------
void check_rng(const Tensor &x, const Tensor &rng, const char *what) {
    if (!rng.defined()) return;
    TORCH_CHECK(rng.scalar_type() == at::kLong && rng.dim() == 1 && rng.size(0) == 2 && rng.is_contiguous(), "loopback_b200.", what,
                ": rng must be a contiguous int64 tensor (seed, offset) or a pair of integers");
    same_device(x, rng, what);
}

Tensor dropout_launch(const Tensor &x, int64_t threshold, const Tensor &rng, int64_t seed, int64_t offset, const Tensor &used) {
    Tensor out = at::empty_like(x);
    On on(x);
    check(lb.lb_dropout(ptr(x), ptr(out), (int)threshold, ptr_as<int64_t>(rng), seed, offset, ptr_as<int64_t>(used), x.numel(), code(x),
                        on.stream), "dropout");
    return out;
}

struct Dropout : torch::autograd::Function<Dropout> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Maybe &rng_, int64_t threshold, int64_t seed, int64_t offset) {
        const Tensor rng = rng_.value_or(Tensor());
        Tensor used = rng.defined() ? at::empty_like(rng) : Tensor();
        Tensor out = dropout_launch(x, threshold, rng, seed, offset, used);
        ctx->save_for_backward({used});
        ctx->saved_data["threshold"] = threshold;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        check_capture("dropout");
        const Tensor used = ctx->get_saved_variables()[0];
        Tensor dx = dropout_launch(dense(g[0]), ctx->saved_data["threshold"].toInt(), used, ctx->saved_data["seed"].toInt(),
                                   ctx->saved_data["offset"].toInt(), Tensor());
        return once({dx, Tensor(), Tensor(), Tensor(), Tensor()}, "dropout");
    }
};

Tensor dropout(const Tensor &x, int64_t threshold, const Maybe &rng, int64_t seed, int64_t offset) {
    TORCH_CHECK(x.is_cuda(), "loopback_b200.dropout: tensors must live on a CUDA device (there is no CPU path)");
    const Tensor pair = rng.value_or(Tensor());
    check_rng(x, pair, "dropout");
    const Tensor xc = dense(x);
    return wants_grad({xc}) ? Dropout::apply(xc, rng, threshold, seed, offset)
                            : dropout_launch(xc, threshold, pair, seed, offset, Tensor());
}

// ---------------------------------------------------------------------------------------------------------
// the end of a block
// ---------------------------------------------------------------------------------------------------------
struct ResidualArgs {
    int kind = LB_GATE_NONE;
    double scale = 1., eps = 0.;
    int64_t threshold = 0, seed = 0, offset = 0;
};

int weight_code(const Tensor &x, const Tensor &w, const Tensor &gate, const Tensor &next_w, int kind) {
    return code(w.defined() ? w : next_w.defined() ? next_w : kind == LB_GATE_CHANNEL ? gate : x);
}

// what the backward wants besides the inputs, in one buffer: the pair dropout used (16 bytes), r_y [n], r_o [n]
variable_list residual_forward(const Tensor &x, const Tensor &y, const Tensor &w, const Tensor &gate, const Tensor &scale,
                               const Tensor &next_w, const Tensor &rng, const ResidualArgs &a, const Tensor &stats) {
    const int64_t d = x.size(-1), n = x.numel() / d;
    Tensor out = at::empty_like(x), u;
    if (next_w.defined()) u = at::empty_like(x);
    float *st = ptr_as<float>(stats);
    On on(x);
    check(lb.lb_residual_fwd(ptr(x), ptr(y), ptr(w), ptr(gate), a.kind, ptr_as<float>(scale), (float)a.scale, ptr(next_w), ptr(out),
                             ptr(u), st && w.defined() ? st + 4 : nullptr, st && u.defined() ? st + 4 + n : nullptr,
                             (int)a.threshold, ptr_as<int64_t>(rng), a.seed, a.offset,
                             st && rng.defined() ? reinterpret_cast<int64_t *>(st) : nullptr, n, (int)d, (float)a.eps, code(x),
                             weight_code(x, w, gate, next_w, a.kind), on.stream), "block residual");
    if (u.defined()) return {out, u};
    return {out};
}

struct BlockResidual : torch::autograd::Function<BlockResidual> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &y, const Maybe &w_, const Maybe &gate_,
                                 const Maybe &scale_, const Maybe &next_w_, const Maybe &rng_, const ResidualArgs *a) {
        const Tensor w = w_.value_or(Tensor()), gate = gate_.value_or(Tensor()), scale = scale_.value_or(Tensor()),
                     next_w = next_w_.value_or(Tensor()), rng = rng_.value_or(Tensor());
        const int64_t n = x.numel() / x.size(-1);
        Tensor stats = floats(4 + 2 * n, x);
        variable_list got = residual_forward(x, y, w, gate, scale, next_w, rng, *a, stats);
        ctx->save_for_backward({x, y, w, gate, scale, next_w, stats});
        ctx->saved_data["kind"] = (int64_t)a->kind;
        ctx->saved_data["scale"] = a->scale;
        ctx->saved_data["threshold"] = a->threshold;
        ctx->saved_data["seed"] = a->seed;
        ctx->saved_data["offset"] = a->offset;
        ctx->saved_data["pair"] = rng.defined();
        ctx->set_materialize_grads(false);
        return got;
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        check_capture("block_residual");
        const variable_list s = ctx->get_saved_variables();
        const Tensor &x = s[0], &y = s[1], &w = s[2], &gate = s[3], &scale = s[4], &next_w = s[5], &stats = s[6];
        const Tensor g_out = g[0].defined() ? dense(g[0]) : Tensor();
        const Tensor g_u = g.size() > 1 && g[1].defined() ? dense(g[1]) : Tensor();
        if (!g_out.defined() && !g_u.defined()) return variable_list(8);
        const int kind = (int)ctx->saved_data["kind"].toInt();
        const int64_t d = x.size(-1), n = x.numel() / d;
        Tensor grad[6];
        for (int i = 0, edge = 0; i < 6; ++i)                     // the node's edges are those of the inputs that are there
            if (s[i].defined() && ctx->needs_input_grad(edge++)) grad[i] = at::empty_like(s[i]);
        Tensor scratch;
        if (grad[2].defined() || grad[4].defined() || grad[5].defined() || (grad[3].defined() && kind == LB_GATE_CHANNEL))
            scratch = bytes(lb.lb_block_scratch_bytes((int)d), x);
        float *st = ptr_as<float>(stats);
        On on(x);
        check(lb.lb_residual_bwd(ptr(x), ptr(y), ptr(w), ptr(gate), kind, ptr_as<float>(scale), (float)ctx->saved_data["scale"].toDouble(),
                                 ptr(next_w), w.defined() ? st + 4 : nullptr, next_w.defined() ? st + 4 + n : nullptr,
                                 (int)ctx->saved_data["threshold"].toInt(),
                                 ctx->saved_data["pair"].toBool() ? reinterpret_cast<int64_t *>(st) : nullptr,
                                 ctx->saved_data["seed"].toInt(), ctx->saved_data["offset"].toInt(), ptr(g_out), ptr(g_u), ptr(grad[0]),
                                 ptr(grad[1]), ptr(grad[2]), ptr(grad[3]), ptr_as<float>(grad[4]), ptr(grad[5]), ptr(scratch), n, (int)d,
                                 code(x), weight_code(x, w, gate, next_w, kind), on.stream), "block residual backward");
        return once({grad[0], grad[1], grad[2], grad[3], grad[4], grad[5], Tensor(), Tensor()}, "block_residual");
    }
};

variable_list block_residual(const Tensor &x, const Tensor &y, const Maybe &weight, const Maybe &gate_,
                             const Maybe &scale_, double scale, const Maybe &next_weight, double eps,
                             int64_t threshold, const Maybe &rng_, int64_t seed, int64_t offset) {
    const char *what = "block_residual";
    require_rows(x, what);
    same_device(x, y, what);
    TORCH_CHECK(y.sizes() == x.sizes() && y.scalar_type() == x.scalar_type(), "loopback_b200.block_residual: x is ", x.sizes(), " ",
                x.scalar_type(), ", y is ", y.sizes(), " ", y.scalar_type());
    Tensor w = weight.value_or(Tensor()), next_w = next_weight.value_or(Tensor()), gate = gate_.value_or(Tensor()), none;
    Tensor scale_t = scale_.value_or(Tensor());
    const Tensor rng = rng_.value_or(Tensor());
    ResidualArgs a;
    if (gate.defined()) {
        same_device(x, gate, what);
        if (gate.dim() == 1 && gate.size(0) == x.size(-1)) a.kind = LB_GATE_CHANNEL;
        else if (gate.sizes() == x.sizes()) a.kind = LB_GATE_FULL;
        else if (gate.dim() == x.dim() && gate.size(-1) == 1 && gate.sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1))
            a.kind = LB_GATE_TOKEN;
        else
            TORCH_CHECK(false, "loopback_b200.block_residual: a gate of shape ", gate.sizes(),
                        " is neither per channel, per token nor per element of ", x.sizes());
        TORCH_CHECK(a.kind == LB_GATE_CHANNEL || gate.scalar_type() == x.scalar_type(),
                    "loopback_b200.block_residual: a gate per token or element has the rows' type, got ", gate.scalar_type());
    }
    channel_params(x, {&w, &next_w, a.kind == LB_GATE_CHANNEL ? &gate : &none}, what);
    if (gate.defined()) gate = dense(gate);
    if (scale_t.defined()) {
        TORCH_CHECK(scale_t.numel() == 1, "loopback_b200.block_residual: a learned scale has one element");
        same_device(x, scale_t, what);
        scale_t = scale_t.to(at::kFloat);
    }
    check_rng(x, rng, what);
    a.scale = scale; a.eps = eps; a.threshold = threshold; a.seed = seed; a.offset = offset;
    const Tensor xc = dense(x), yc = dense(y);
    if (wants_grad({xc, yc, w, gate, scale_t, next_w})) {
        const auto maybe = [](const Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); };
        return BlockResidual::apply(xc, yc, maybe(w), maybe(gate), maybe(scale_t), maybe(next_w), maybe(rng), &a);
    }
    return residual_forward(xc, yc, w, gate, scale_t, next_w, rng, a, none);
}

// ---------------------------------------------------------------------------------------------------------
// the gated feed-forward block
// ---------------------------------------------------------------------------------------------------------
Tensor ffn_workspace(int64_t n, int64_t d, int64_t f, int kind, const Tensor &like) {
    const size_t need = lb.lb_ffn_workspace_bytes(n, (int)d, (int)f, kind);
    TORCH_CHECK(need > 0, "loopback_b200.gated_ffn: ", lb.lb_last_error_string());
    return bytes(need, like);
}

Tensor ffn_forward(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t act, const Tensor &h, const Tensor &kept) {
    const int64_t d = x.size(-1), f = wg.size(0), n = x.numel() / d;
    Tensor y = at::empty_like(x);
    On on(x);
    const Tensor ws = ffn_workspace(n, d, f, h.defined() ? LB_FFN_FORWARD : LB_FFN_INFERENCE, x);
    check(lb.lb_ffn_fwd(ptr(x), ptr(wg), ptr(wu), ptr(wd), ptr(y), ptr(h), ptr(kept), ptr(ws), (size_t)ws.numel(), n, (int)d, (int)f,
                        (int)act, LB_DTYPE_BF16, on.stream), "gated ffn");
    return y;
}

struct GatedFFN : torch::autograd::Function<GatedFFN> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t act) {
        const int64_t f = wg.size(0), n = x.numel() / x.size(-1);
        Tensor h = at::empty({n, f}, x.options());
        Tensor kept = bytes(lb.lb_ffn_kept_bytes(n, (int)f), x);
        Tensor y = ffn_forward(x, wg, wu, wd, act, h, kept);
        ctx->save_for_backward({x, wg, wu, wd, h, kept});
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        check_capture("gated_ffn");
        const variable_list s = ctx->get_saved_variables();
        const Tensor &x = s[0], &wg = s[1], &wu = s[2], &wd = s[3], &h = s[4], &kept = s[5];
        const int64_t d = x.size(-1), f = wg.size(0), n = x.numel() / d;
        const Tensor dy = dense(g[0]);
        const bool need_g = ctx->needs_input_grad(1), need_u = ctx->needs_input_grad(2);
        Tensor dx, dgu, dwd;
        if (ctx->needs_input_grad(0)) dx = at::empty_like(x);
        if (need_g || need_u) dgu = at::empty({2, f, d}, x.options());
        if (ctx->needs_input_grad(3)) dwd = at::empty_like(wd);
        On on(x);
        const Tensor ws = ffn_workspace(n, d, f, LB_FFN_BACKWARD, x);
        check(lb.lb_ffn_bwd(ptr(x), ptr(wg), ptr(wu), ptr(wd), ptr(h), ptr(kept), ptr(dy), ptr(dx), ptr(dgu), ptr(dwd), ptr(ws),
                            (size_t)ws.numel(), n, (int)d, (int)f, LB_DTYPE_BF16, on.stream), "gated ffn backward");
        return once({dx, need_g ? dgu[0] : Tensor(), need_u ? dgu[1] : Tensor(), dwd, Tensor()}, "gated_ffn");
    }
};

Tensor gated_ffn(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t act) {
    const char *what = "gated_ffn";
    require_rows(x, what);
    for (const Tensor *w : {&wg, &wu, &wd}) same_device(x, *w, what);
    const int64_t d = x.size(-1);
    TORCH_CHECK(wg.dim() == 2 && wg.size(1) == d && wu.sizes() == wg.sizes() && wd.dim() == 2 && wd.size(0) == d && wd.size(1) == wg.size(0),
                "loopback_b200.gated_ffn: rows have ", d, " columns, weights are ", wg.sizes(), ", ", wu.sizes(), ", ", wd.sizes(),
                "; expected (f, d), (f, d), (d, f)");
    for (const Tensor *t : std::initializer_list<const Tensor *>{&x, &wg, &wu, &wd})
        TORCH_CHECK(t->scalar_type() == at::kBFloat16, "loopback_b200.gated_ffn: the products run in bf16, got ", t->scalar_type());
    for (const Tensor *w : {&wg, &wu, &wd}) TORCH_CHECK(w->is_contiguous(), "loopback_b200.gated_ffn: weights must be contiguous");
    TORCH_CHECK(d < (1 << 30) && wg.size(0) < (1 << 30), "loopback_b200.gated_ffn: d=", d, ", f=", wg.size(0), " are too large");
    const Tensor xc = dense(x);
    return wants_grad({xc, wg, wu, wd}) ? GatedFFN::apply(xc, wg, wu, wd, act) : ffn_forward(xc, wg, wu, wd, act, Tensor(), Tensor());
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
    m.def("bind", &bind);
    m.def("block_norm", &block_norm);
    m.def("dropout", &dropout);
    m.def("block_residual", &block_residual);
    m.def("gated_ffn", &gated_ffn);
}
