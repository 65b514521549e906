// jq_torch.cpp -- the policy operators as torch functions with gradients
// (module junqi_b200._policy): argument checks, outputs from torch's allocator,
// the current stream of the tensors' device, and autograd nodes.  The kernels
// are the library's; their entry points come from `bind`, so this module and
// the ctypes binding share one loaded library.
//
// It is C++ because a training step's small calls are bound by the host: with
// the nodes in Python a forward and backward pass of a layer norm took 121 us
// on the host whatever its size, here 67 (torch's own takes 70); a sampling
// call 34, here 8.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ExpandUtils.h>
#include <ATen/ops/clamp.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/jq.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

struct Api {
    decltype(&jq_last_error) last_error;
    decltype(&jq_layer_norm) layer_norm;
    decltype(&jq_layer_norm_scratch_floats) layer_norm_scratch;
    decltype(&jq_layer_norm_backward) layer_norm_backward;
    decltype(&jq_action_log_prob) log_prob;
    decltype(&jq_action_log_prob_backward) log_prob_backward;
    decltype(&jq_verify_drafts) verify;
} api{};

void bind(const std::unordered_map<std::string, uintptr_t> &at) {
    api.last_error = reinterpret_cast<decltype(api.last_error)>(at.at("jq_last_error"));
    api.layer_norm = reinterpret_cast<decltype(api.layer_norm)>(at.at("jq_layer_norm"));
    api.layer_norm_scratch = reinterpret_cast<decltype(api.layer_norm_scratch)>(at.at("jq_layer_norm_scratch_floats"));
    api.layer_norm_backward = reinterpret_cast<decltype(api.layer_norm_backward)>(at.at("jq_layer_norm_backward"));
    api.log_prob = reinterpret_cast<decltype(api.log_prob)>(at.at("jq_action_log_prob"));
    api.log_prob_backward = reinterpret_cast<decltype(api.log_prob_backward)>(at.at("jq_action_log_prob_backward"));
    api.verify = reinterpret_cast<decltype(api.verify)>(at.at("jq_verify_drafts"));
}

#define REQUIRE(COND, ...)                                             \
    do {                                                               \
        if (!(COND)) throw py::value_error(c10::str(__VA_ARGS__));     \
    } while (0)

void check(int status, const char *what) {
    if (status == JQ_OK) return;
    static const char *const names[] = {"", "JQ_ERR_ARG", "JQ_ERR_CUDA", "JQ_ERR_NOT_READY", "JQ_ERR_CAPACITY"};
    throw std::runtime_error(c10::str(what, " failed: ", status > 0 && status < 5 ? names[status] : "?", ": ", api.last_error()));
}

std::string shape_of(at::IntArrayRef s) {  // as Python writes a tuple
    std::string t = "(";
    for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
    return t + (s.size() == 1 ? ",)" : ")");
}

int dtype_of(const char *what, const Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return JQ_F32;
        case at::kHalf: return JQ_F16;
        case at::kBFloat16: return JQ_BF16;
        default: REQUIRE(false, what, " must be float32, float16 or bfloat16, got ", t.scalar_type()); return -1;
    }
}

void same_device(const char *what, const Tensor &x, std::initializer_list<const Tensor *> others) {
    for (const Tensor *t : others)
        if (t->defined()) REQUIRE(t->device() == x.device(), what, ": tensors on ", x.device(), " and ", t->device());
    REQUIRE(x.is_cuda(), what, ": needs CUDA tensors, got ", x.device());
}

// Forward-mode derivatives are not given: a tangent would be lost without a word.
void no_tangent(const char *what, std::initializer_list<const Tensor *> inputs) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor *t : inputs)
        REQUIRE(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), what, " has no forward-mode derivative");
}

// `t` as its memory has it: the imaginary part of a conjugate is negated only when torch reads it.
Tensor read(const Tensor &t) { return t.is_neg() ? t.resolve_neg() : t; }

// `t` with neighbouring places next to each other on its last axis.
Tensor last(const Tensor &t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? read(t) : t.contiguous(); }
// (rows, n) view (a copy only where the leading axes have no common stride).
Tensor rows_of(const Tensor &t) { return last(t.dim() == 2 ? t : t.reshape({-1, t.size(-1)})); }
// The same inside a node's forward pass, where views have no history: with it, so that `once` finds the way back to `t`.
Tensor saved_rows_of(const Tensor &t) {
    at::AutoGradMode history(true);
    return rows_of(t);
}

// `t` as contiguous int32 of `shape`; 64-bit values are cut to [lo, hi] first, so that none wraps.
Tensor ints(const char *what, const Tensor &t, at::IntArrayRef shape, int64_t lo, int64_t hi) {
    const auto k = t.scalar_type();
    REQUIRE(k == at::kInt || k == at::kLong || k == at::kShort || k == at::kChar || k == at::kByte, what, " must be whole numbers, got ", t.scalar_type());
    REQUIRE(t.sizes() == shape, what, " must be ", shape_of(shape), ", got ", shape_of(t.sizes()));
    if (t.scalar_type() == at::kInt) return t.contiguous();
    return (t.scalar_type() == at::kLong ? t.clamp(lo, hi) : t).to(at::kInt).contiguous();
}

Tensor uniform(const char *what, const Tensor &u, at::IntArrayRef shape) {
    REQUIRE(u.scalar_type() == at::kFloat && u.sizes() == shape, what, " must be float32 ", shape_of(shape), ", got ",
            u.scalar_type(), " ", shape_of(u.sizes()));
    return read(u).contiguous();
}

// The mask, expanded to `shape`; undefined without one.
Tensor mask_for(const char *what, const MaybeTensor &mask, at::IntArrayRef shape) {
    if (!mask) return {};
    REQUIRE(mask->scalar_type() == at::kByte || mask->scalar_type() == at::kBool, what, ": the mask must be uint8 or bool, got ",
            mask->scalar_type());
    REQUIRE(at::is_expandable_to(mask->sizes(), shape), what, ": a mask of ", shape_of(mask->sizes()), " does not fit logits of ",
            shape_of(shape));
    return mask->sizes() == shape ? *mask : mask->expand(shape);
}

int64_t actions_of(const char *what, const Tensor &logits, int64_t dim) {
    dtype_of(c10::str(what, ": logits").c_str(), logits);
    REQUIRE(logits.dim() >= 1 && (dim == 0 || logits.dim() == dim), what, ": logits of ", shape_of(logits.sizes()));
    const int64_t n = logits.size(-1);
    REQUIRE(n > 0 && n <= JQ_POLICY_MAX_ACTIONS, what, ": 1 to ", JQ_POLICY_MAX_ACTIONS, " actions, got ", n);
    return n;
}

template <typename T = void>
T *ptr(const Tensor &t) { return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr; }

// The tensors' device made current, and its current stream.
struct On {
    c10::cuda::CUDAGuard guard;
    void *stream;
    explicit On(const Tensor &t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.get_device()).stream()) {}
};

// Gradients that are asked for with create_graph depend on `from`, but their own differentiation is an error.
variable_list once(variable_list out, const variable_list &from) {
    if (!at::GradMode::is_enabled()) return out;
    auto node = std::make_shared<torch::autograd::Error>("the policy operators are differentiable once",
                                                         torch::autograd::collect_next_edges(from));
    for (auto &t : out)
        if (t.defined()) torch::autograd::set_history(t, node);
    return out;
}

// ---- layer norm --------------------------------------------------------------

Tensor norm_forward(const Tensor &x, const Tensor &x2, const Tensor &weight, const Tensor &bias, double eps, const Tensor &stats) {
    Tensor y = at::empty(x.sizes(), x.options());
    if (x2.size(0) > 0) {
        On on(x);
        const Tensor &w = weight.defined() ? weight : bias;
        check(api.layer_norm(ptr(x2), x2.stride(0), ptr(weight), ptr(bias), x2.size(0), (int32_t)x2.size(1), dtype_of("x", x),
                             w.defined() ? dtype_of("weight", w) : JQ_F32, (float)eps, ptr(y), ptr<float>(stats), on.stream),
              "jq_layer_norm");
    }
    return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const MaybeTensor &w, const MaybeTensor &b, double eps) {
        const Tensor weight = w.value_or(Tensor()), bias = b.value_or(Tensor());
        const Tensor x2 = saved_rows_of(x), stats = at::empty({x2.size(0), 3}, x.options().dtype(at::kFloat));
        ctx->save_for_backward({x2, weight, bias, stats});
        return norm_forward(x, x2, weight, bias, eps, stats);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x2 = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3], &dy = grads[0];
        const int64_t rows = x2.size(0), dim = x2.size(1);
        Tensor dx, dw, db, scratch;
        if (dy.defined()) {
            at::NoGradGuard no_grad;
            // (inputs are counted without those that were not given)
            if (ctx->needs_input_grad(0)) dx = at::empty(dy.sizes(), x2.options());
            if (weight.defined() && ctx->needs_input_grad(1)) dw = at::empty({dim}, weight.options());
            if (bias.defined() && ctx->needs_input_grad(weight.defined() ? 2 : 1)) db = at::empty({dim}, bias.options());
            if (rows > 0) {
                On on(x2);
                const Tensor dy2 = rows_of(dy), &w = weight.defined() ? weight : bias;
                if (dw.defined() || db.defined())
                    scratch = at::empty({api.layer_norm_scratch(rows, (int32_t)dim)}, x2.options().dtype(at::kFloat));
                check(api.layer_norm_backward(ptr(x2), x2.stride(0), ptr(weight), ptr(dy2), dy2.stride(0), ptr<float>(stats), rows,
                                              (int32_t)dim, dtype_of("x", x2), w.defined() ? dtype_of("weight", w) : JQ_F32,
                                              ptr(dx), ptr(dw), ptr(db), ptr<float>(scratch), on.stream),
                      "jq_layer_norm_backward");
            } else {
                if (dw.defined()) dw.zero_();
                if (db.defined()) db.zero_();
            }
        }
        return once({dx, dw, db, Tensor()}, {x2, weight, dy});
    }
};

Tensor layer_norm(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &bias, double eps) {
    dtype_of("layer_norm: x", x);
    REQUIRE(x.dim() > 0 && x.size(-1) > 0, "layer_norm: x needs a last axis, got ", shape_of(x.sizes()));
    REQUIRE(x.size(-1) <= INT32_MAX, "layer_norm: a last axis of ", x.size(-1));
    REQUIRE(eps >= 0, "layer_norm: eps must not be negative, got ", std::to_string(eps));
    const int64_t dim = x.size(-1);
    const std::pair<const char *, const MaybeTensor *> given[] = {{"weight", &weight}, {"bias", &bias}};
    for (const auto &[name, p] : given) {
        if (!*p) continue;
        const Tensor &t = **p;
        REQUIRE(t.dim() == 1 && t.size(0) == dim, "layer_norm: ", name, " must be ", shape_of({dim}), ", got ", shape_of(t.sizes()));
        REQUIRE(t.scalar_type() == at::kFloat || t.scalar_type() == x.scalar_type(), "layer_norm: ", name,
                " must be float32 or ", x.scalar_type(), ", got ", t.scalar_type());
    }
    REQUIRE(!weight || !bias || weight->scalar_type() == bias->scalar_type(), "layer_norm: weight and bias must have one type");
    no_tangent("layer_norm", {&x, weight ? &*weight : &x, bias ? &*bias : &x});
    const Tensor w = weight ? read(*weight).contiguous() : Tensor(), b = bias ? read(*bias).contiguous() : Tensor();
    same_device("layer_norm", x, {&w, &b});
    if (at::GradMode::is_enabled() && (x.requires_grad() || (weight && weight->requires_grad()) || (bias && bias->requires_grad())))
        return LayerNorm::apply(x, weight ? MaybeTensor(w) : MaybeTensor(), bias ? MaybeTensor(b) : MaybeTensor(), eps);
    at::NoGradGuard no_grad;
    return norm_forward(x, rows_of(x), w, b, eps, Tensor());
}

// ---- log-probability and entropy -----------------------------------------------

std::pair<Tensor, Tensor> logp_forward(const Tensor &logits, const Tensor &x2, const Tensor &m2, const Tensor &act, const Tensor &stats,
                                       const Tensor &bits) {
    const auto shape = logits.sizes().slice(0, logits.dim() - 1);
    const auto options = logits.options().dtype(at::kFloat);
    Tensor lp = at::empty(shape, options), ent = at::empty(shape, options);
    if (x2.size(0) > 0) {
        On on(logits);
        check(api.log_prob(ptr(x2), x2.stride(0), dtype_of("logits", x2), ptr<uint8_t>(m2), m2.defined() ? m2.stride(0) : 0,
                           ptr<int32_t>(act), x2.size(0), (int32_t)x2.size(1), ptr<float>(lp), ptr<float>(ent), ptr<float>(stats),
                           ptr<uint32_t>(bits), on.stream),
              "jq_action_log_prob");
    }
    return {lp, ent};
}

struct ActionLogProb : torch::autograd::Function<ActionLogProb> {
    static variable_list forward(AutogradContext *ctx, const Tensor &logits, const MaybeTensor &mask, const Tensor &act) {
        const Tensor x2 = saved_rows_of(logits), m2 = mask ? rows_of(*mask) : Tensor();
        const int64_t rows = x2.size(0), n = x2.size(1);
        const Tensor stats = at::empty({rows, 4}, logits.options().dtype(at::kFloat));
        const Tensor bits = mask ? at::empty({rows, (n + 31) / 32}, logits.options().dtype(at::kInt)) : Tensor();
        ctx->save_for_backward({x2, stats, bits});
        ctx->set_materialize_grads(false);
        auto [lp, ent] = logp_forward(logits, x2, m2, act, stats, bits);
        return {lp, ent};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x2 = saved[0], &stats = saved[1], &bits = saved[2];
        const Tensor &some = grads[0].defined() ? grads[0] : grads[1];
        if (!some.defined()) return {Tensor(), Tensor(), Tensor()};
        Tensor dx;
        {
            at::NoGradGuard no_grad;
            auto shape = some.sizes().vec();
            shape.push_back(x2.size(1));
            dx = at::empty(shape, x2.options());
            if (x2.size(0) > 0) {
                On on(x2);
                const Tensor u = grads[0].defined() ? read(grads[0]).reshape({-1}) : Tensor(), v = grads[1].defined() ? read(grads[1]).reshape({-1}) : Tensor();
                check(api.log_prob_backward(ptr(x2), x2.stride(0), dtype_of("logits", x2), ptr<uint32_t>(bits),
                                            ptr<float>(stats), ptr<float>(u), u.defined() ? u.stride(0) : 0, ptr<float>(v),
                                            v.defined() ? v.stride(0) : 0, x2.size(0), (int32_t)x2.size(1), ptr(dx), on.stream),
                      "jq_action_log_prob_backward");
            }
        }
        return once({dx, Tensor(), Tensor()}, {x2, grads[0], grads[1]});
    }
};

std::pair<Tensor, Tensor> action_log_prob(const Tensor &logits, const MaybeTensor &mask, const Tensor &actions) {
    const int64_t n = actions_of("action_log_prob", logits, 0);
    const Tensor act = ints("action_log_prob: actions", actions, logits.sizes().slice(0, logits.dim() - 1), -1, n);
    const Tensor m = mask_for("action_log_prob", mask, logits.sizes());
    no_tangent("action_log_prob", {&logits});
    same_device("action_log_prob", logits, {&m, &act});
    if (at::GradMode::is_enabled() && logits.requires_grad()) {
        auto out = ActionLogProb::apply(logits, m.defined() ? MaybeTensor(m) : MaybeTensor(), act);
        return {out[0], out[1]};
    }
    at::NoGradGuard no_grad;
    return logp_forward(logits, rows_of(logits), m.defined() ? rows_of(m) : Tensor(), act, Tensor(), Tensor());
}

// ---- sampling and verification ----------------------------------------------------

std::tuple<Tensor, Tensor, Tensor> verify(const Tensor &x, const Tensor &drafts, const Tensor &accept_u, const Tensor &sample_u,
                                          const Tensor &y, const Tensor &mask, const Tensor &lengths, at::IntArrayRef shape) {
    const int64_t games = x.size(0), places = x.size(1);
    REQUIRE(games <= INT32_MAX, "too many games: ", games);
    const auto whole = x.options().dtype(at::kInt);
    Tensor out = at::empty(shape, whole), lp = at::empty(shape, x.options().dtype(at::kFloat)), acc = at::empty({games}, whole);
    if (games > 0) {
        On on(x);
        jq_drafts d{};
        d.games = (int32_t)games, d.drafts = (int32_t)(places - 1), d.actions = (int32_t)x.size(2), d.dtype = dtype_of("logits", x);
        d.logits = ptr(x), d.logits_game = x.stride(0), d.logits_place = x.stride(1);
        if (y.defined()) d.draft_logits = ptr(y), d.draft_game = y.stride(0), d.draft_place = y.stride(1);
        if (mask.defined()) d.mask = ptr<uint8_t>(mask), d.mask_game = mask.stride(0), d.mask_place = mask.stride(1);
        d.drafted = ptr<int32_t>(drafts), d.lengths = ptr<int32_t>(lengths), d.accept_u = ptr<float>(accept_u);
        d.sample_u = ptr<float>(sample_u), d.accepted = ptr<int32_t>(acc), d.out_actions = ptr<int32_t>(out);
        d.log_probs = ptr<float>(lp);
        check(api.verify(&d, on.stream), "jq_verify_drafts");
    }
    return {acc, out, lp};
}

std::tuple<Tensor, Tensor, Tensor> verify_drafts(const Tensor &logits, const Tensor &drafts, const Tensor &accept_u,
                                                 const Tensor &sample_u, const MaybeTensor &draft_logits, const MaybeTensor &mask,
                                                 const MaybeTensor &lengths) {
    at::NoGradGuard no_grad;
    const int64_t n = actions_of("verify_drafts", logits, 3), games = logits.size(0), places = logits.size(1);
    REQUIRE(places >= 1 && places <= JQ_POLICY_MAX_DRAFTS + 1, "verify_drafts: 1 to ", JQ_POLICY_MAX_DRAFTS + 1, " places a game, got ", places);
    const Tensor a = ints("verify_drafts: drafts", drafts, {games, places - 1}, -1, n);
    const Tensor u = uniform("verify_drafts: accept_u", accept_u, {games, places - 1}), r = uniform("verify_drafts: sample_u", sample_u, {games});
    Tensor y, len;
    if (draft_logits) {
        const int64_t want[] = {games, places - 1, n};
        REQUIRE(draft_logits->scalar_type() == logits.scalar_type() && draft_logits->sizes() == at::IntArrayRef(want),
                "verify_drafts: draft_logits must be ", logits.scalar_type(), " ", shape_of(want), ", got ", draft_logits->scalar_type(),
                " ", shape_of(draft_logits->sizes()));
        y = last(*draft_logits);
    }
    if (lengths) len = ints("verify_drafts: lengths", *lengths, {games}, 0, places - 1);
    const Tensor m = mask_for("verify_drafts", mask, logits.sizes());
    same_device("verify_drafts", logits, {&a, &u, &r, &y, &m, &len});
    return verify(last(logits), a, u, r, y, m.defined() ? last(m) : m, len, {games, places});
}

std::pair<Tensor, Tensor> sample_actions(const Tensor &logits, const MaybeTensor &mask, const Tensor &u) {
    at::NoGradGuard no_grad;
    actions_of("sample_actions", logits, 0);
    const auto shape = logits.sizes().slice(0, logits.dim() - 1);
    const Tensor r = uniform("sample_actions: u", u, shape), m = mask_for("sample_actions", mask, logits.sizes());
    same_device("sample_actions", logits, {&m, &r});
    auto [acc, out, lp] = verify(rows_of(logits).unsqueeze(1), Tensor(), Tensor(), r, Tensor(),
                                 m.defined() ? rows_of(m).unsqueeze(1) : m, Tensor(), shape);
    return {out, lp};
}

}  // namespace

PYBIND11_MODULE(_policy, m) {
    m.attr("built_for") = "junqi_b200 built for " JQ_BUILT_FOR;
    const auto free = py::call_guard<py::gil_scoped_release>();
    m.def("bind", &bind);
    m.def("layer_norm", &layer_norm, free);
    m.def("action_log_prob", &action_log_prob, free);
    m.def("verify_drafts", &verify_drafts, free);
    m.def("sample_actions", &sample_actions, free);
}
