// Token embedding and vocabulary cross entropy as autograd nodes: allocation, layout and streams on torch's side, everything else behind the
// C entries (include/trajnet_hip.h).
//
// A node in C++: the engine runs the backward pass of device tensors on a thread of its own, and a Python node costs that thread the
// interpreter lock and cold bytecode (1000 x 64 into 4099 rows, forward and backward: 90 us against 46; the engine alone, for a product with a constant, takes 41).
//
// The entries come as addresses from the library that the package has loaded, so this file links against torch alone.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/trajnet_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Entries {
    decltype(&tnp_last_error) last_error;
    decltype(&tnp_token_embedding_forward) embed_forward;
    decltype(&tnp_token_embedding_backward_workspace_bytes) embed_workspace;
    decltype(&tnp_token_embedding_backward) embed_backward;
    decltype(&tnp_vocab_ce_saved_bytes) ce_saved;
    decltype(&tnp_vocab_ce_workspace_bytes) ce_workspace;
    decltype(&tnp_vocab_ce_forward) ce_forward;
    decltype(&tnp_vocab_ce_backward) ce_backward;
} entry;
static_assert(sizeof(Entries) == 8 * sizeof(void *), "addresses in the order of bind()");

void bind(const std::vector<uint64_t> &addresses) {
    TORCH_CHECK(addresses.size() == 8, "bind: eight addresses");
    memcpy(&entry, addresses.data(), sizeof(entry));
}

void check(int rc, const char *what) { TORCH_CHECK(rc == 0, what, " failed (", rc, "): ", entry.last_error()); }

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int dtype_of(const Tensor &t) {
    return t.scalar_type() == at::kFloat ? TNP_F32 : t.scalar_type() == at::kBFloat16 ? TNP_BF16 : TNP_F16;
}

Tensor workspace(size_t bytes, const Tensor &like) { return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)); }
void *data(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// sizes that the entries take as 32 bits: one that does not fit is refused there
int32_t narrow(int64_t n) { return (int32_t)std::min<int64_t>(n, INT32_MAX); }

// a tangent would be dropped in silence
void no_tangent(const Tensor &t) { TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "the vocabulary operators have no forward-mode derivative"); }

// rows with unit column stride that do not overlap; a copy only where the layout asks for one
struct Rows {
    Tensor t;
    int64_t ld;
    explicit Rows(const Tensor &in) : t(in), ld(in.size(-1)) {
        if (t.is_contiguous()) return;
        if (t.dim() == 2 && t.stride(1) == 1 && t.stride(0) >= ld) ld = t.stride(0);
        else t = t.contiguous();
    }
};

// ---- token embedding ----------------------------------------------------------------------------------------------------------
Tensor embedding_forward(const Tensor &tokens, const Tensor &weight, double scale) {
    const c10::DeviceGuard guard(weight.device());
    const Rows w(weight);
    const Tensor tok = tokens.contiguous();
    const int64_t v = weight.size(0), d = weight.size(1);
    std::vector<int64_t> shape = tokens.sizes().vec();
    shape.push_back(d);
    Tensor out = at::empty(shape, weight.options());
    check(entry.embed_forward(tok.data_ptr(), (int)tok.element_size(), tok.numel(), w.t.data_ptr(), w.ld, v, narrow(d), dtype_of(weight),
                              (float)scale, out.data_ptr(), d, stream_of(weight)), "tnp_token_embedding_forward");
    return out;
}

Tensor embedding_backward(const Tensor &grad, const Tensor &tokens, int64_t entries, double scale) {
    const c10::DeviceGuard guard(grad.device());
    const Rows g(grad);
    const Tensor tok = tokens.contiguous();
    const int64_t n = tok.numel(), d = grad.size(-1);
    Tensor dw = at::empty({entries, d}, grad.options()), ws;
    const size_t need = entry.embed_workspace(n, entries, narrow(d));
    if (need) ws = workspace(need, grad);
    check(entry.embed_backward(tok.data_ptr(), (int)tok.element_size(), n, g.t.data_ptr(), g.ld, entries, narrow(d), dtype_of(grad), (float)scale,
                               dw.data_ptr(), d, data(ws), need, stream_of(grad)), "tnp_token_embedding_backward");
    return dw;
}

// Gradients have no gradient: where one is asked for (create_graph), they are tied to what they were made of by a node that raises.
struct Raise : torch::autograd::Function<Raise> {
    typedef const std::optional<Tensor> &Maybe;
    static Tensor forward(AutogradContext *, const Tensor &grad, Maybe, Maybe, Maybe, Maybe) { return grad.detach(); }
    static variable_list backward(AutogradContext *, const variable_list &) {
        TORCH_CHECK(false, "the gradient of a vocabulary operator has no gradient");
    }
};
variable_list once(variable_list grads, const variable_list &made_of) {
    if (!at::GradMode::is_enabled()) return grads;
    std::optional<Tensor> of[4];
    for (size_t k = 0; k < made_of.size() && k < 4; ++k)
        if (made_of[k].defined()) of[k] = made_of[k];
    for (Tensor &t : grads)
        if (t.defined()) t = Raise::apply(t, of[0], of[1], of[2], of[3]);
    return grads;
}

struct EmbeddingNode : torch::autograd::Function<EmbeddingNode> {
    static Tensor forward(AutogradContext *ctx, const Tensor &tokens, const Tensor &weight, double scale) {
        ctx->save_for_backward({tokens});
        ctx->saved_data["entries"] = weight.size(0);
        ctx->saved_data["scale"] = scale;
        return embedding_forward(tokens, weight, scale);
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        return once({Tensor(), embedding_backward(grads[0], ctx->get_saved_variables()[0], ctx->saved_data["entries"].toInt(),
                                                  ctx->saved_data["scale"].toDouble()), Tensor()}, grads);
    }
};

Tensor token_embedding(const Tensor &tokens, const Tensor &weight, double scale) {
    no_tangent(weight);
    if (weight.requires_grad() && at::GradMode::is_enabled()) return EmbeddingNode::apply(tokens, weight, scale);
    return embedding_forward(tokens, weight, scale);
}

// ---- cross entropy over a vocabulary ------------------------------------------------------------------------------------------
struct CeArgs {
    Tensor t, b;
    tnp_vocab_ce c = {};
    CeArgs(const Tensor &weight, const Tensor &target, const Tensor &bias, int64_t reduction)
        : t(target.to(at::kLong).contiguous()), b(bias.defined() ? bias.contiguous() : bias) {
        c.dtype = dtype_of(weight);
        c.reduction = (int32_t)reduction;
        c.M = t.numel();
        c.V = narrow(weight.size(0));
        c.D = narrow(weight.size(1));
        c.ld_hidden = c.ld_weight = weight.size(1);
        c.bias = data(b);
        c.target = t.data_ptr<int64_t>();
    }
};

// (loss, what the backward pass reads: undefined where none will follow); at least one row
std::pair<Tensor, Tensor> ce_forward(const Tensor &hidden, const Tensor &weight, const Tensor &target, const Tensor &bias, int64_t reduction,
                                     bool train) {
    const c10::DeviceGuard guard(weight.device());
    CeArgs a(weight, target, bias, reduction);
    const Rows x(hidden), w(weight);
    a.c.hidden = x.t.data_ptr();
    a.c.ld_hidden = x.ld;
    a.c.weight = w.t.data_ptr();
    a.c.ld_weight = w.ld;
    Tensor saved;
    if (train) {
        saved = workspace(entry.ce_saved(&a.c), weight);
        a.c.saved = saved.data_ptr();
    }
    const size_t need = entry.ce_workspace(&a.c, 0);
    const Tensor ws = workspace(need, weight);
    Tensor loss = at::empty(reduction == 0 ? target.sizes() : at::IntArrayRef(), weight.options().dtype(at::kFloat));
    check(entry.ce_forward(&a.c, loss.data_ptr<float>(), ws.data_ptr(), need, stream_of(weight)), "tnp_vocab_ce_forward");
    return {loss, saved};
}

variable_list ce_backward(const Tensor &grad, const Tensor &hidden, const Tensor &weight, const Tensor &target, const Tensor &bias,
                          const Tensor &saved, int64_t reduction, bool need_x, bool need_w, bool need_b) {
    const c10::DeviceGuard guard(weight.device());
    CeArgs a(weight, target, bias, reduction);                  // hidden states and weight are read from what was saved
    a.c.saved = saved.data_ptr();
    const Tensor g = grad.to(at::kFloat).contiguous();
    Tensor dx, dw, db;
    if (need_x) dx = at::empty(hidden.sizes(), hidden.options());
    if (need_w) dw = at::empty(weight.sizes(), weight.options());
    if (need_b) db = at::empty(bias.sizes(), bias.options());
    const size_t need = entry.ce_workspace(&a.c, 1);
    const Tensor ws = workspace(need, weight);
    check(entry.ce_backward(&a.c, g.data_ptr<float>(), data(dx), data(dw), data(db), ws.data_ptr(), need, stream_of(weight)),
          "tnp_vocab_ce_backward");
    return {dx, dw, db};
}

Tensor or_undefined(const std::optional<Tensor> &t) { return t ? *t : Tensor(); }

struct CeNode : torch::autograd::Function<CeNode> {
    static Tensor forward(AutogradContext *ctx, const Tensor &hidden, const Tensor &weight, const std::optional<Tensor> &bias,
                          const Tensor &target, int64_t reduction) {
        const Tensor b = or_undefined(bias);
        auto [loss, saved] = ce_forward(hidden, weight, target, b, reduction, true);
        ctx->save_for_backward({hidden, weight, b, target, saved});
        ctx->saved_data["reduction"] = reduction;
        return loss;
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        const variable_list s = ctx->get_saved_variables();
        variable_list d = ce_backward(grads[0], s[0], s[1], s[3], s[2], s[4], ctx->saved_data["reduction"].toInt(), ctx->needs_input_grad(0),
                                      ctx->needs_input_grad(1), s[2].defined() && ctx->needs_input_grad(2));
        d.resize(5);
        return once(std::move(d), {grads[0], s[0], s[1], s[2]});
    }
};

Tensor vocab_cross_entropy(const Tensor &hidden, const Tensor &weight, const Tensor &target, const std::optional<Tensor> &bias,
                           int64_t reduction) {
    const Tensor b = or_undefined(bias);
    for (const Tensor &t : {hidden, weight, b}) no_tangent(t);
    if (at::GradMode::is_enabled() && (hidden.requires_grad() || weight.requires_grad() || (b.defined() && b.requires_grad())))
        return CeNode::apply(hidden, weight, bias, target, reduction);
    return ce_forward(hidden, weight, target, b, reduction, false).first;
}

}  // namespace

PYBIND11_MODULE(_trajnet_torch, m) {
    m.def("bind", &bind);
    m.def("token_embedding", &token_embedding);
    m.def("embedding_forward", &embedding_forward);
    m.def("embedding_backward", &embedding_backward);
    m.def("vocab_cross_entropy", &vocab_cross_entropy);
    m.def("ce_forward", [](const Tensor &hidden, const Tensor &weight, const Tensor &target, const std::optional<Tensor> &bias, int64_t reduction) {
        return ce_forward(hidden, weight, target, or_undefined(bias), reduction, true);
    });
    m.def("ce_backward", [](const Tensor &grad, const Tensor &hidden, const Tensor &weight, const Tensor &target, const std::optional<Tensor> &bias,
                            const Tensor &saved, int64_t reduction) {
        const Tensor b = or_undefined(bias);
        const variable_list d = ce_backward(grad, hidden, weight, target, b, saved, reduction, true, true, b.defined());
        return std::make_tuple(d[0], d[1], d[2]);
    });
}
