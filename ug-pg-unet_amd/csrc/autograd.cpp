// Autograd nodes of the group norm and the distillation loss (and the call that records a
// teacher's top logits), over libugpg's C entries.
//
// A backward pass runs on the autograd engine's device thread.  Python there is dear: every
// object it shares with the calling thread moves between two cores, so that a small training
// pass through a Python autograd.Function took 81-97 us of which the engine itself is 43 (an
// elementwise product and its gradient).  These nodes keep Python out of the backward.
// Arguments are checked by the Python callers (ugpg/norm.py, ugpg/distill.py); the entries are
// bound at import by address, so this module runs the very library ugpg._C loaded.
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <unordered_set>
#include <vector>

#include "../../include/ugpg.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

struct Entries {
    decltype(&ugpg_last_error) last_error = nullptr;
    decltype(&ugpg_group_norm_workspace) gn_ws = nullptr;
    decltype(&ugpg_group_norm_fwd) gn_fwd = nullptr;
    decltype(&ugpg_group_norm_bwd) gn_bwd = nullptr;
    decltype(&ugpg_distill_workspace) ds_ws = nullptr;
    decltype(&ugpg_distill_fwd) ds_fwd = nullptr;
    decltype(&ugpg_distill_bwd) ds_bwd = nullptr;
    decltype(&ugpg_top_logits) top = nullptr;
} lib;

void bind(const std::vector<uintptr_t>& at) {
    TORCH_CHECK(at.size() == 8, "ugpg autograd: 8 entries expected");
    lib.last_error = reinterpret_cast<decltype(lib.last_error)>(at[0]);
    lib.gn_ws = reinterpret_cast<decltype(lib.gn_ws)>(at[1]);
    lib.gn_fwd = reinterpret_cast<decltype(lib.gn_fwd)>(at[2]);
    lib.gn_bwd = reinterpret_cast<decltype(lib.gn_bwd)>(at[3]);
    lib.ds_ws = reinterpret_cast<decltype(lib.ds_ws)>(at[4]);
    lib.ds_fwd = reinterpret_cast<decltype(lib.ds_fwd)>(at[5]);
    lib.ds_bwd = reinterpret_cast<decltype(lib.ds_bwd)>(at[6]);
    lib.top = reinterpret_cast<decltype(lib.top)>(at[7]);
}

void check(int rc, const char* what) {
    TORCH_CHECK(rc == 0, "ugpg ", what, " failed (", rc, "): ", lib.last_error());
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
int dtype_of(const Tensor& t) { return t.scalar_type() == torch::kFloat ? UGPG_DT_F32 : UGPG_DT_BF16; }
const float* floats(const Maybe& t) { return t.has_value() && t->defined() ? t->data_ptr<float>() : nullptr; }
Maybe some(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }
Tensor scratch(size_t bytes, const Tensor& like) {
    return torch::empty({(int64_t)bytes}, like.options().dtype(torch::kByte));
}

// A graph capture must not take in a node of the default stream: its backward would make that
// stream, which cannot be captured, wait on the captured one, and the process ends.  An
// input's node, or a leaf's accumulator while an eager graph of the same leaf lives, is one.
void check_capture(const char* what, std::initializer_list<const Tensor*> inputs) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    for (const Tensor* t : inputs) {
        if (!t->defined() || !t->requires_grad()) continue;
        const auto node = t->grad_fn() ? t->grad_fn() : torch::autograd::impl::try_get_grad_accumulator(*t);
        const auto s = node ? node->stream() : std::nullopt;
        TORCH_CHECK(!s || s->id() != 0, what, ": captured while a graph of the same input lives on the "
                    "default stream; drop that graph first, or run it on another stream");
    }
}

// The same for what lies behind this node: a captured backward that is about to run into a node of
// the default stream (a view or a cast of a leaf whose eager graph lives, say) ends here, with
// an error, while that stream is untouched.  Only nodes that this pass executes count.
void check_captured_backward(const char* what) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const auto self = torch::autograd::get_current_node();
    const auto* info = torch::autograd::get_current_graph_task_exec_info();  // empty: all execute
    std::unordered_set<torch::autograd::Node*> seen;
    std::vector<torch::autograd::Node*> todo;
    if (self) todo.push_back(self.get());
    while (!todo.empty()) {
        torch::autograd::Node* const node = todo.back();
        todo.pop_back();
        for (const auto& edge : node->next_edges()) {
            torch::autograd::Node* const next = edge.function.get();
            if (!next || !seen.insert(next).second) continue;
            if (info && !info->empty()) {
                const auto it = info->find(next);
                if (it == info->end() || !it->second.should_execute()) continue;
            }
            const auto s = next->stream();
            TORCH_CHECK(!s || s->id() != 0, what, ": its backward is captured while a graph of the same "
                        "input lives on the default stream; drop that graph first, or run it on another stream");
            todo.push_back(next);
        }
    }
}

// A tangent of forward-mode differentiation would be left out of the result: refused, for
// constants of a loss too.  (Undefined wherever forward mode is off.)
void check_tangents(const char* what, std::initializer_list<const Tensor*> inputs) {
    for (const Tensor* t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), what,
                                    ": forward-mode derivatives are not implemented");
}

// The gradients of a backward that runs with create_graph: differentiating through one of them
// raises, whether or not the upstream gradient required one.
void once(const char* what, variable_list& grads) {
    if (!c10::GradMode::is_enabled()) return;
    variable_list live;
    for (auto& g : grads)
        if (g.defined()) live.push_back(g.detach().requires_grad_(true));
    auto err = std::make_shared<torch::autograd::DelayedError>(
        std::string(what) + " can be differentiated only once", (int64_t)live.size());
    variable_list out = (*err)(std::move(live));
    size_t k = 0;
    for (auto& g : grads)
        if (g.defined()) g = out[k++];
}

// ---------------------------------------------------------------- group norm
ugpg_group_norm_t gn_desc(const Tensor& x, int64_t groups, const Maybe& w, const Maybe& b, double eps,
                          int64_t act, const Tensor& stats) {
    ugpg_group_norm_t d{};
    const int64_t B = x.size(0), C = x.size(-1);
    d.x = x.data_ptr();
    d.dtype = dtype_of(x);
    d.B = (int)B;
    d.HW = x.numel() / (B * C);
    d.C = (int)C;
    d.G = (int)groups;
    d.gamma = floats(w);
    d.beta = floats(b);
    d.eps = (float)eps;
    d.act = (int)act;
    d.mean = stats.data_ptr<float>();
    d.rstd = d.mean + B * groups;
    return d;
}

// y; `stats` [2][B][groups] receives the means and reciprocal deviations
Tensor gn_forward(const Tensor& x, int64_t groups, const Maybe& w, const Maybe& b, double eps, int64_t act,
                  Tensor& stats) {
    c10::OptionalDeviceGuard guard(x.device());
    Tensor y = torch::empty_like(x);
    stats = torch::empty({2, x.size(0), groups}, x.options().dtype(torch::kFloat));
    const ugpg_group_norm_t d = gn_desc(x, groups, w, b, eps, act, stats);
    const size_t n = lib.gn_ws(&d, 0);
    const Tensor ws = scratch(n, x);
    check(lib.gn_fwd(&d, y.data_ptr(), ws.data_ptr(), n, stream_of(x)), "group_norm_fwd");
    return y;
}

struct GroupNormAct : torch::autograd::Function<GroupNormAct> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& w, const Maybe& b, int64_t groups,
                          double eps, int64_t act) {
        Tensor stats;
        Tensor y = gn_forward(x, groups, w, b, eps, act, stats);
        ctx->save_for_backward({x, w.value_or(Tensor()), b.value_or(Tensor()), stats});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["act"] = act;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list up) {
        const variable_list s = ctx->get_saved_variables();  // (raises if one was written in place since)
        const Tensor &x = s[0], &w = s[1], &b = s[2];
        c10::OptionalDeviceGuard guard(x.device());
        check_captured_backward("group_norm_act");
        const Tensor dy = up[0].detach().to(x.scalar_type()).contiguous();
        const ugpg_group_norm_t d = gn_desc(x, ctx->saved_data["groups"].toInt(), some(w), some(b), 0.0,
                                            ctx->saved_data["act"].toInt(), s[3]);
        Tensor dx = torch::empty_like(x), dw, db;
        size_t edge = 1;  // (an absent weight or bias has no edge)
        if (w.defined() && ctx->needs_input_grad(edge++)) dw = torch::empty_like(w);
        if (b.defined() && ctx->needs_input_grad(edge)) db = torch::empty_like(b);
        const size_t n = lib.gn_ws(&d, 1);
        const Tensor ws = scratch(n, x);
        check(lib.gn_bwd(&d, dy.data_ptr(), d.dtype, dx.data_ptr(), d.dtype,
                         dw.defined() ? dw.data_ptr<float>() : nullptr,
                         db.defined() ? db.data_ptr<float>() : nullptr, nullptr, ws.data_ptr(), n, stream_of(x)),
              "group_norm_bwd");
        variable_list g{dx, dw, db};
        once("group_norm_act", g);
        if (!ctx->needs_input_grad(0)) g[0] = Tensor();
        return {g[0], g[1], g[2], Tensor(), Tensor(), Tensor()};
    }
};

bool wants(const Maybe& t) { return t.has_value() && t->defined() && t->requires_grad(); }

Tensor group_norm_act(const Tensor& x, const Maybe& w, const Maybe& b, int64_t groups, double eps, int64_t act) {
    const Tensor none;
    check_tangents("group_norm_act", {&x, w ? &*w : &none, b ? &*b : &none});
    if (c10::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b))) {
        check_capture("group_norm_act", {&x, w ? &*w : &none, b ? &*b : &none});
        return GroupNormAct::apply(x, w, b, groups, eps, act);
    }
    Tensor stats;
    c10::AutoGradMode off(false);
    return gn_forward(x, groups, w, b, eps, act, stats);
}

// ---------------------------------------------------------------- distillation
// rows of any row stride and unit column stride, or packed class maps; else a copy
Tensor class_rows(const Tensor& z) {
    const int64_t N = z.size(0), V = z.size(1);
    if (z.numel() > N * V) return z.contiguous();
    Tensor r = z.reshape({N, V});
    const bool ok = (V == 1 || r.stride(1) == 1) && (N == 1 || r.stride(0) >= V);
    return ok ? r : r.contiguous();
}

ugpg_distill_t ds_desc(const Tensor& shape, const Tensor& z, const Tensor& values, const Tensor& indices,
                       const Maybe& rest, const Maybe& weight, double T, double scale) {
    ugpg_distill_t d{};
    d.logits = z.data_ptr();
    d.dtype = dtype_of(z);
    d.N = shape.size(0);
    d.V = (int)shape.size(1);
    d.inner = shape.numel() / (d.N * d.V);
    d.stride = d.inner > 1 ? (int64_t)d.V * d.inner : std::max<int64_t>(z.stride(0), d.V);
    d.values = values.data_ptr();
    d.values_dtype = dtype_of(values);
    d.indices = indices.data_ptr();
    d.index_bits = indices.scalar_type() == torch::kInt ? 32 : 64;
    d.k = (int)values.size(1);
    d.rest = floats(rest);
    d.weight = floats(weight);
    d.temperature = T;
    d.scale = scale;
    return d;
}

Tensor ds_forward(const Tensor& logits, const Tensor& values, const Tensor& indices, const Maybe& rest,
                  const Maybe& weight, double T, double scale, bool per_row, Tensor* dz) {
    c10::OptionalDeviceGuard guard(logits.device());
    const Tensor z = class_rows(logits.detach());
    const ugpg_distill_t d = ds_desc(logits, z, values, indices, rest, weight, T, scale);
    std::vector<int64_t> lead;
    if (per_row) {
        lead = logits.sizes().vec();
        lead.erase(lead.begin() + 1);
    }
    Tensor loss = torch::empty(lead, logits.options().dtype(torch::kFloat));
    if (dz) *dz = torch::empty(logits.sizes(), logits.options());
    const size_t n = lib.ds_ws(&d, 0);
    const Tensor ws = scratch(n, logits);
    float* out = loss.data_ptr<float>();
    check(lib.ds_fwd(&d, per_row ? nullptr : out, per_row ? out : nullptr, dz ? dz->data_ptr() : nullptr,
                     ws.data_ptr(), n, stream_of(logits)),
          "distill_fwd");
    return loss;
}

struct Distill : torch::autograd::Function<Distill> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& values,
                          const Tensor& indices, const Maybe& rest, const Maybe& weight, double T,
                          double scale, bool per_row) {
        // A scalar loss writes its gradient here, for an upstream gradient of 1, while each row
        // is in the caches: one reading of the logits instead of two.
        Tensor dz;
        Tensor loss = ds_forward(logits, values, indices, rest, weight, T, scale, per_row,
                                 per_row ? nullptr : &dz);
        ctx->save_for_backward({logits, values, indices, rest.value_or(Tensor()), weight.value_or(Tensor())});
        ctx->saved_data["T"] = T;
        ctx->saved_data["scale"] = scale;
        if (!per_row) ctx->saved_data["dz"] = dz;
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list up) {
        const variable_list s = ctx->get_saved_variables();  // (raises if one was written in place since)
        const Tensor& logits = s[0];
        c10::OptionalDeviceGuard guard(logits.device());
        check_captured_backward("distillation_loss");
        const Tensor z = class_rows(logits.detach());
        const ugpg_distill_t d = ds_desc(logits, z, s[1], s[2], some(s[3]), some(s[4]),
                                         ctx->saved_data["T"].toDouble(), ctx->saved_data["scale"].toDouble());
        const Tensor gout = up[0].detach().to(torch::kFloat).contiguous();
        Tensor dz;
        const auto it = ctx->saved_data.find("dz");
        const bool ready = it != ctx->saved_data.end();
        if (ready) {  // handed out once; a second backward writes its own
            dz = it->second.toTensor();
            ctx->saved_data.erase(it);
        } else {
            dz = torch::empty(logits.sizes(), logits.options());
        }
        const size_t n = lib.ds_ws(&d, 1);
        const Tensor ws = n ? scratch(n, logits) : Tensor();
        check(lib.ds_bwd(&d, gout.data_ptr<float>(), gout.dim() > 0, ready, dz.data_ptr(),
                         n ? ws.data_ptr() : nullptr, n, stream_of(logits)),
              "distill_bwd");
        variable_list g{dz};
        once("distillation_loss", g);
        return {g[0], Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor distill(const Tensor& logits, const Tensor& values, const Tensor& indices, const Maybe& rest,
               const Maybe& weight, double T, double scale, bool per_row) {
    const Tensor none;
    check_tangents("distillation_loss", {&logits, &values, rest ? &*rest : &none, weight ? &*weight : &none});
    if (c10::GradMode::is_enabled() && logits.requires_grad()) {
        check_capture("distillation_loss", {&logits});
        return Distill::apply(logits, values, indices, rest, weight, T, scale, per_row);
    }
    c10::AutoGradMode off(false);
    return ds_forward(logits, values, indices, rest, weight, T, scale, per_row, nullptr);
}

// values, indices [N][k][*spatial] and the rest's logit [N][*spatial]; no gradient
std::vector<Tensor> top_logits(const Tensor& logits, int64_t k, double T) {
    c10::AutoGradMode off(false);
    c10::OptionalDeviceGuard guard(logits.device());
    const Tensor z = class_rows(logits.detach());
    const int64_t N = logits.size(0), V = logits.size(1), inner = logits.numel() / (N * V);
    std::vector<int64_t> rec = logits.sizes().vec(), lead = rec;
    rec[1] = k;
    lead.erase(lead.begin() + 1);
    const Tensor values = torch::empty(rec, logits.options());
    const Tensor indices = torch::empty(rec, logits.options().dtype(torch::kLong));
    const Tensor rest = torch::empty(lead, logits.options().dtype(torch::kFloat));
    check(lib.top(z.data_ptr(), dtype_of(z), N, (int)V, inner,
                  inner > 1 ? V * inner : std::max<int64_t>(z.stride(0), V), (int)k, (float)T, values.data_ptr(),
                  indices.data_ptr<int64_t>(), rest.data_ptr<float>(), stream_of(z)),
          "top_logits");
    return {values, indices, rest};
}

}  // namespace

#ifndef UGPG_AUTOGRAD_ID
#define UGPG_AUTOGRAD_ID ""
#endif

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    typedef py::call_guard<py::gil_scoped_release> nogil;
    m.attr("build_id") = UGPG_AUTOGRAD_ID;
    m.def("bind", &bind);
    m.def("group_norm_act", &group_norm_act, nogil());
    m.def("distill", &distill, nogil());
    m.def("top_logits", &top_logits, nogil());
}
