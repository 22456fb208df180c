// ops_torch.cpp -- the operators of include/ccsp_ops.h on torch tensors: argument checks, allocation, streams, autograd (the Python side is operators.py).
// Host code only; the kernels are libccsp_ops.so's.  It exists because a call is short: the smallest operators run 3 us on the GPU, and what
// a call costs its host -- checks, allocations, the autograd node -- is what a user waits for (in Python: 14 us a call, 50 us with its gradient).
#include <c10/hip/HIPStream.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include "../../../include/ccsp_ops.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<Tensor> MaybeTensor;

PyObject* g_ccsp_error = nullptr;      // diffusion_ccsp_amd.CcspError, held by the module
struct OpsError : std::runtime_error { using std::runtime_error::runtime_error; };

template <typename... A> std::string text(const A&... a) { return c10::str(a...); }
#define VALUE(cond, ...) do { if (!(cond)) throw py::value_error(text(__VA_ARGS__)); } while (0)
#define TYPE(cond, ...) do { if (!(cond)) throw py::type_error(text(__VA_ARGS__)); } while (0)
void run(int rc) { if (rc != 0) throw OpsError(ccsp_ops_last_error()); }

int type_code(at::ScalarType t) { return t == at::kFloat ? CCSP_OPS_F32 : (t == at::kBFloat16 ? CCSP_OPS_BF16 : (t == at::kHalf ? CCSP_OPS_F16 : -1)); }
int code(const Tensor& t) { return type_code(t.scalar_type()); }
std::string name_of(const Tensor& t) {                           // a type as Python spells it
    const auto s = t.scalar_type();
    return s == at::kFloat ? "float32" : s == at::kDouble ? "float64" : s == at::kHalf ? "float16" : s == at::kBFloat16 ? "bfloat16" : s == at::kInt ? "int32" : s == at::kLong ? "int64" : c10::toString(s);
}

// the library works on the current device: this one, for the scope of a call
struct On {
    c10::DeviceGuard guard;
    void* stream;
    explicit On(const Tensor& t) : guard(t.device()), stream((void*)c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

// (a trace records torch's own operations: of a kernel, nothing but the memory that its result goes to)
void not_recorded(const char* who) {
    if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY) || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch))
        throw OpsError(text(who, ": cannot be recorded by torch.jit.trace or make_fx; it may be captured into a graph of the GPU's"));
}

// what every tensor of a call has to be
void usable(const char* who, const Tensor& t) {
    // (a tangent would be lost without a word: the kernels read the values alone)
    if (t._fw_grad(0).defined()) throw OpsError(text(who, ": forward-mode derivatives are not supported; gradients come through torch.autograd in reverse"));
    // (a wrapper -- a distributed or quantised tensor, one inside torch.func's transforms -- has no memory of its own)
    TYPE(t.layout() == at::kStrided, who, ": a tensor that is sparse or blocked; supported are dense ones");
    TYPE(t.has_storage() && (!t.unsafeGetTensorImpl()->is_python_dispatch() || t.unsafeGetTensorImpl()->unsafe_storage().unsafeGetStorageImpl()->_mutable_data_ptr_no_checks().get()), who,
         ": a tensor that wraps others (a subclass without memory, a transform's); supported are plain ones");
    if (!t.is_cuda()) throw OpsError(text(who, ": tensors must be on a GPU (got ", t.device(), "); there is no CPU fallback"));
}
void same_device(const char* who, const Tensor& a, const Tensor& b) { VALUE(a.device() == b.device(), who, ": tensors on ", a.device(), " and ", b.device()); }

// a view that stands for the negative of its memory, or for zeros without memory
bool lazy(const Tensor& t) { return t.is_neg() || t._is_zerotensor(); }
Tensor whole(const Tensor& t) { return lazy(t) ? t.clone(at::MemoryFormat::Contiguous) : t.contiguous(); }
// a matrix the kernels can read: last dimension contiguous
Tensor rows_of(const Tensor& t) { return !lazy(t) && (t.size(1) <= 1 || t.stride(1) == 1) ? t : whole(t); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// What route() leaves on the device: one int32 tensor with everything in it.
struct Plan {
    Tensor buf;
    int64_t n_experts = 0, n_tokens = 0, n_rows = 0, k = 0;
    bool listed = false;
    std::vector<int64_t> shape;
    enum { OFFSETS, ROWS, ASSIGN, ROW_TOKEN, PLACE, TOKEN_PTR, TOKEN_ASSIGN, END };
    int64_t at(int which) const {                                // first element of a part
        const int64_t a = n_experts + 1, o[8] = {0, a, a + n_rows, a + 2 * n_rows, a + 3 * n_rows, a + 4 * n_rows, a + 4 * n_rows + n_tokens + 1, a + 5 * n_rows + n_tokens + 1};
        return which == END && !listed ? o[TOKEN_PTR] : o[which];
    }
    int32_t* p(int which) const { return buf.data_ptr<int32_t>() + at(which); }
    Tensor view(int which, int64_t n) const { return buf.narrow(0, at(which), n); }
    int32_t* token_order() const { return listed ? p(TOKEN_ASSIGN) : nullptr; }
    Tensor offsets() const { return view(OFFSETS, n_experts + 1); }
    Tensor rows() const { return view(ROWS, n_rows); }
    Tensor assign() const { return view(ASSIGN, n_rows); }
    Tensor row_token() const { return view(ROW_TOKEN, n_rows); }
    MaybeTensor token_ptr() const { return listed ? MaybeTensor(view(TOKEN_PTR, n_tokens + 1)) : MaybeTensor(); }
    MaybeTensor token_assign() const { return listed ? MaybeTensor(view(TOKEN_ASSIGN, n_rows)) : MaybeTensor(); }
    Tensor counts() const { return offsets().diff(); }
    // what an autograd node keeps of a plan
    void save(AutogradContext* c) const { c->saved_data["plan"] = std::vector<int64_t>{n_experts, n_tokens, n_rows, k, listed}; }
    static Plan load(AutogradContext* c, const Tensor& buf) {
        const auto v = c->saved_data["plan"].toIntVector();
        Plan q;
        q.buf = buf; q.n_experts = v[0]; q.n_tokens = v[1]; q.n_rows = v[2]; q.k = v[3]; q.listed = v[4];
        return q;
    }
};

std::shared_ptr<Plan> route(const Tensor& expert_in, int64_t n_experts, const MaybeTensor& tokens_in, c10::optional<int64_t> n_tokens) {
    not_recorded("route");
    usable("route", expert_in);
    TYPE(expert_in.scalar_type() == at::kInt || expert_in.scalar_type() == at::kLong, "route: expert ids must be int32 or int64, got ", name_of(expert_in));
    VALUE(n_experts >= 1 && n_experts <= CCSP_OPS_MAX_EXPERTS, "route: ", n_experts, " experts, supported are 1 to ", CCSP_OPS_MAX_EXPERTS);
    auto q = std::make_shared<Plan>();
    Tensor tokens;
    if (!tokens_in) {
        VALUE(expert_in.dim() == 1 || expert_in.dim() == 2, "route: expert ids must be [N] or [N, k], got ", expert_in.sizes());
        VALUE(!n_tokens || *n_tokens == expert_in.size(0), "route: ", n_tokens.value_or(0), " tokens, but expert ids of ", expert_in.size(0));
        q->n_tokens = expert_in.size(0);
        q->k = expert_in.dim() == 1 ? 1 : expert_in.size(1);
        VALUE(q->k > 0, "route: no expert per token");
    } else {
        usable("route", *tokens_in);
        same_device("route", expert_in, *tokens_in);
        VALUE(tokens_in->sizes() == expert_in.sizes() && tokens_in->scalar_type() == expert_in.scalar_type(), "route: tokens ", name_of(*tokens_in), " ", tokens_in->sizes(),
              " and expert ids ", name_of(expert_in), " ", expert_in.sizes(), " differ");
        VALUE(n_tokens && *n_tokens >= 0, "route: tokens need n_tokens");
        q->n_tokens = *n_tokens;
        q->listed = true;
        tokens = whole(*tokens_in);
    }
    const Tensor expert = whole(expert_in);
    q->n_experts = n_experts;
    q->n_rows = expert.numel();
    q->shape = expert.sizes().vec();
    const int64_t need = ccsp_ops_route_workspace(q->n_rows, (int32_t)n_experts, q->n_tokens, q->listed);
    VALUE(need >= 0, "route: ", q->n_rows, " assignments of ", q->n_tokens, " tokens are out of range");
    On on(expert);
    q->buf = at::empty({q->at(Plan::END)}, expert.options().dtype(at::kInt));
    const Tensor ws = at::empty({need}, expert.options().dtype(at::kByte));
    run(ccsp_ops_route(ptr(expert), ptr(tokens), (int32_t)expert.element_size() * 8, q->n_rows, (int32_t)q->k, (int32_t)n_experts, q->n_tokens, q->p(Plan::OFFSETS), q->p(Plan::ROWS),
                       q->p(Plan::ASSIGN), q->p(Plan::ROW_TOKEN), q->p(Plan::PLACE), q->listed ? q->p(Plan::TOKEN_PTR) : nullptr, q->token_order(), ptr(ws), need, on.stream));
    return q;
}

Tensor gather(const Tensor& src_in, const Plan& q) {
    On on(src_in);
    const Tensor src = rows_of(src_in), out = at::empty({q.n_rows, src.size(1)}, src.options());
    run(ccsp_ops_rows_gather(code(src), q.n_rows, src.size(1), ptr(src), src.stride(0), q.p(Plan::ROW_TOKEN), q.p(Plan::ASSIGN), q.p(Plan::PLACE), q.token_order(), ptr(out), on.stream));
    return out;
}

Tensor combine(const Tensor& src_in, const Plan& q, const Tensor& weights) {
    On on(src_in);
    const Tensor src = rows_of(src_in), out = at::empty({q.n_tokens, src.size(1)}, src.options());
    run(ccsp_ops_rows_combine(code(src), q.n_tokens, q.n_rows, src.size(1), (int32_t)q.k, q.listed ? q.p(Plan::TOKEN_PTR) : nullptr, q.token_order(), q.p(Plan::ROWS), ptr(weights),
                              weights.defined() ? code(weights) : CCSP_OPS_F32, ptr(src), src.stride(0), ptr(out), on.stream));
    return out;
}

// Gradients of gradients are refused where they would be used: with a graph of the backward pass asked for (`more`), a gradient's own gradient is an error.
variable_list first_order(const char* who, bool more, variable_list g) {
    if (!more) return g;
    at::AutoGradMode on(true);
    for (auto& t : g)
        if (t.defined()) t = (*std::make_shared<torch::autograd::DelayedError>(text(who, " is differentiable once"), 1))({t.detach().set_requires_grad(true)})[0];
    return g;
}
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

struct SortRows : torch::autograd::Function<SortRows> {
    static Tensor forward(AutogradContext* c, const Tensor& x, const Tensor& buf, const Plan* q) {
        q->save(c);
        c->save_for_backward({buf});
        return gather(x, *q);
    }
    static variable_list backward(AutogradContext* c, variable_list g) {
        const bool more = at::GradMode::is_enabled();
        at::NoGradGuard no;
        not_recorded("sort_rows");
        usable("sort_rows", g[0]);
        const Plan q = Plan::load(c, c->get_saved_variables()[0]);
        return first_order("sort_rows", more, {combine(g[0], q, Tensor()), Tensor(), Tensor()});
    }
};

struct CombineRows : torch::autograd::Function<CombineRows> {
    // (an absent tensor is an absent optional: it has no edge in the graph, so needs_input_grad counts past it, to the plan's, which is false)
    static Tensor forward(AutogradContext* c, const Tensor& ys, const MaybeTensor& given, const Tensor& buf, const Plan* q) {
        const Tensor weights = given.value_or(Tensor());
        q->save(c);
        c->save_for_backward({buf, wants_grad(weights) ? ys : Tensor(), weights});
        return combine(ys, *q, weights);
    }
    static variable_list backward(AutogradContext* c, variable_list grads) {
        const bool more = at::GradMode::is_enabled();
        at::NoGradGuard no;
        not_recorded("combine_rows");
        usable("combine_rows", grads[0]);
        const auto saved = c->get_saved_variables();
        const Plan q = Plan::load(c, saved[0]);
        const Tensor& weights = saved[2];
        if (!weights.defined()) return first_order("combine_rows", more, {gather(grads[0], q), Tensor(), Tensor(), Tensor()});
        const bool want_ys = c->needs_input_grad(0), want_w = c->needs_input_grad(1);
        const Tensor g = rows_of(grads[0]), ys = want_w ? rows_of(saved[1]) : Tensor();
        On on(g);
        const Tensor d_ys = want_ys ? at::empty({q.n_rows, g.size(1)}, g.options()) : Tensor(), d_w = want_w ? at::empty(weights.sizes(), weights.options()) : Tensor();
        run(ccsp_ops_rows_back(code(g), q.n_rows, g.size(1), q.p(Plan::ROW_TOKEN), q.p(Plan::ASSIGN), q.p(Plan::PLACE), q.token_order(), ptr(weights), code(weights), ptr(g), g.stride(0), ptr(ys), want_w ? ys.stride(0) : 0, ptr(d_ys), ptr(d_w),
                               on.stream));
        return first_order("combine_rows", more, {d_ys, d_w, Tensor(), Tensor()});
    }
};

void float_rows(const char* who, const char* name, const Tensor& t, int64_t n, const char* what) {
    VALUE(t.dim() == 2 && t.size(0) == n, who, ": ", name, " must be [", n, ", width] (", what, "), got ", t.sizes());
    TYPE(code(t) >= 0, who, ": ", name, " of type ", name_of(t), "; supported are float32, bfloat16 and float16");
    VALUE(t.size(1) <= CCSP_OPS_MAX_WIDTH, who, ": ", name, " of width ", t.size(1), " is out of range");
}

Tensor sort_rows(const Tensor& x, const Plan& q) {
    not_recorded("sort_rows");
    usable("sort_rows", x);
    same_device("sort_rows", x, q.buf);
    float_rows("sort_rows", "x", x, q.n_tokens, "one row per token");
    if (at::GradMode::is_enabled() && x.requires_grad()) return SortRows::apply(x, q.buf, &q);
    return gather(x, q);
}

Tensor combine_rows(const Tensor& ys, const Plan& q, const MaybeTensor& weights_in) {
    not_recorded("combine_rows");
    usable("combine_rows", ys);
    same_device("combine_rows", ys, q.buf);
    float_rows("combine_rows", "ys", ys, q.n_rows, "one row per assignment");
    Tensor weights;
    if (weights_in) {
        usable("combine_rows", *weights_in);
        same_device("combine_rows", ys, *weights_in);
        VALUE(weights_in->sizes() == at::IntArrayRef(q.shape), "combine_rows: weights ", weights_in->sizes(), " for expert ids ", at::IntArrayRef(q.shape));
        TYPE(weights_in->scalar_type() == at::kFloat || weights_in->scalar_type() == ys.scalar_type(), "combine_rows: weights of type ", name_of(*weights_in), " for rows of type ",
             name_of(ys), "; supported are float32 and the rows' type");
        weights = whole(*weights_in);
    }
    if (at::GradMode::is_enabled() && (ys.requires_grad() || wants_grad(weights))) return CombineRows::apply(ys, weights.defined() ? MaybeTensor(weights) : MaybeTensor(), q.buf, &q);
    return combine(ys, q, weights);
}

// a product's workspace
struct Space {
    Tensor t;
    int64_t bytes;
    Space(int product, const Tensor& a, const Tensor& b, const Plan& q, int64_t O, int64_t I) {
        bytes = ccsp_ops_linear_workspace(product, code(a), (int32_t)q.n_experts, q.n_rows, I, O, ptr(a), a.stride(0), ptr(b), b.stride(-2));
        if (bytes < 0) throw OpsError(text("expert_linear: ", ccsp_ops_last_error()));
        if (bytes > 0) t = at::empty({bytes}, a.options().dtype(at::kByte));
    }
};

Tensor linear_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Plan& q, int64_t act, Tensor* z) {
    On on(x);
    const int64_t O = weight.size(1), I = weight.size(2);
    const Tensor y = at::empty({q.n_rows, O}, x.options());
    if (z) *z = at::empty({q.n_rows, O}, x.options());
    const Space ws(CCSP_OPS_FORWARD, x, weight, q, O, I);
    run(ccsp_ops_linear(code(x), (int32_t)q.n_experts, q.n_rows, I, O, q.p(Plan::OFFSETS), ptr(x), x.stride(0), ptr(weight), ptr(bias), (int32_t)act, ptr(y), z ? ptr(*z) : nullptr, ptr(ws.t), ws.bytes,
                        on.stream));
    return y;
}

struct ExpertLinear : torch::autograd::Function<ExpertLinear> {
    static Tensor forward(AutogradContext* c, const Tensor& xs, const Tensor& weight, const MaybeTensor& given, const Tensor& buf, const Plan* q, int64_t act) {
        const Tensor bias = given.value_or(Tensor());
        const Tensor x = rows_of(xs);
        Tensor z;
        const Tensor y = linear_forward(x, weight, bias, *q, act, act ? &z : nullptr);
        q->save(c);
        c->saved_data["act"] = act;
        c->save_for_backward({buf, wants_grad(weight) || wants_grad(bias) ? x : Tensor(), weight, z});
        return y;
    }
    static variable_list backward(AutogradContext* c, variable_list grads) {
        const bool more = at::GradMode::is_enabled();
        at::NoGradGuard no;
        not_recorded("expert_linear");
        usable("expert_linear", grads[0]);
        const auto saved = c->get_saved_variables();
        const Plan q = Plan::load(c, saved[0]);
        const Tensor &x = saved[1], &weight = saved[2], &z = saved[3];
        const int64_t O = weight.size(1), I = weight.size(2);
        const int32_t E = (int32_t)q.n_experts;
        Tensor dz = rows_of(grads[0]), d_x, d_w, d_b;
        On on(dz);
        const int type = code(dz);
        if (c->saved_data["act"].toInt()) {
            const Tensor g = dz;
            dz = at::empty({q.n_rows, O}, g.options());
            run(ccsp_ops_linear_silu_back(type, E, q.n_rows, O, q.p(Plan::OFFSETS), ptr(g), g.stride(0), ptr(z), ptr(dz), on.stream));
        }
        if (c->needs_input_grad(0)) {
            d_x = at::empty({q.n_rows, I}, dz.options());
            const Space ws(CCSP_OPS_BACK_INPUT, dz, weight, q, O, I);
            run(ccsp_ops_linear_back_input(type, E, q.n_rows, I, O, q.p(Plan::OFFSETS), ptr(dz), dz.stride(0), ptr(weight), ptr(d_x), ptr(ws.t), ws.bytes, on.stream));
        }
        const bool want_w = c->needs_input_grad(1), want_b = c->needs_input_grad(2);
        if (want_w || want_b) {
            if (want_w) d_w = at::empty({E, O, I}, dz.options());
            if (want_b) d_b = at::empty({E, O}, dz.options());
            const Space ws(CCSP_OPS_BACK_WEIGHT, dz, x, q, O, I);
            run(ccsp_ops_linear_back_weight(type, E, q.n_rows, I, O, q.p(Plan::OFFSETS), ptr(dz), dz.stride(0), ptr(x), x.stride(0), ptr(d_w), ptr(d_b), ptr(ws.t), ws.bytes, on.stream));
        }
        return first_order("expert_linear", more, {d_x, d_w, d_b, Tensor(), Tensor(), Tensor()});
    }
};

Tensor expert_linear(const Tensor& xs, const Tensor& weight_in, const Plan& q, const MaybeTensor& bias_in, const c10::optional<std::string>& activation) {
    not_recorded("expert_linear");
    usable("expert_linear", xs);
    usable("expert_linear", weight_in);
    same_device("expert_linear", xs, q.buf);
    same_device("expert_linear", xs, weight_in);
    float_rows("expert_linear", "xs", xs, q.n_rows, "one row per assignment");
    VALUE(!activation || *activation == "silu", "expert_linear: activation '", activation.value_or(""), "'; supported are None and 'silu'");
    VALUE(weight_in.dim() == 3 && weight_in.size(0) == q.n_experts && weight_in.size(2) == xs.size(1) && weight_in.size(1) > 0 && weight_in.size(2) > 0, "expert_linear: weight must be [",
          q.n_experts, ", out, ", xs.size(1), "], got ", weight_in.sizes());
    VALUE(weight_in.size(1) <= CCSP_OPS_MAX_FEATURES && weight_in.size(2) <= CCSP_OPS_MAX_FEATURES, "expert_linear: weight ", weight_in.sizes(), " is out of range");
    Tensor bias;
    if (bias_in) {
        usable("expert_linear", *bias_in);
        same_device("expert_linear", xs, *bias_in);
        VALUE(bias_in->dim() == 2 && bias_in->size(0) == weight_in.size(0) && bias_in->size(1) == weight_in.size(1), "expert_linear: bias must be [", weight_in.size(0), ", ", weight_in.size(1),
              "], got ", bias_in->sizes());
        bias = whole(*bias_in);
    }
    TYPE(weight_in.scalar_type() == xs.scalar_type() && (!bias.defined() || bias.scalar_type() == xs.scalar_type()), "expert_linear: xs, weight and bias must have one type, got ",
         name_of(xs), ", ", name_of(weight_in), bias.defined() ? text(", ", name_of(bias)) : "");
    const Tensor weight = whole(weight_in);
    const int64_t act = activation ? CCSP_OPS_SILU : CCSP_OPS_NONE;
    if (at::GradMode::is_enabled() && (xs.requires_grad() || weight.requires_grad() || wants_grad(bias))) return ExpertLinear::apply(xs, weight, bias.defined() ? MaybeTensor(bias) : MaybeTensor(), q.buf, &q, act);
    return linear_forward(rows_of(xs), weight, bias, q, act, nullptr);
}

// norm of the tensors; max_norm: and the tensors scaled, in place or into `out`
Tensor clip(const std::string& name, const std::vector<Tensor>& src, c10::optional<double> max_norm, const c10::optional<std::vector<Tensor>>& out) {
    const char* who = name.c_str();
    VALUE(!src.empty(), who, ": no tensors");
    VALUE(src.size() < (1u << 30), who, ": too many tensors");
    VALUE(!max_norm || *max_norm >= 0, who, ": max_norm ", max_norm.value_or(0), " must not be negative");
    VALUE(!out || out->size() == src.size(), who, ": out must hold one tensor of the same type and shape per gradient");
    const size_t n = src.size();
    std::vector<Tensor> hold;                                    // contiguous copies; in place, `back` says where they go
    std::vector<size_t> back;
    std::vector<const void*> from(n);
    std::vector<void*> to(n);
    std::vector<int64_t> sizes(n);
    std::vector<int32_t> types(n);
    not_recorded(who);
    usable(who, src[0]);
    On on(src[0]);
    at::NoGradGuard no;
    for (size_t i = 0; i < n; ++i) {
        const Tensor& t = src[i];
        usable(who, t);
        VALUE(t.device() == src[0].device(), who, ": tensors on ", src[0].device(), " and ", t.device());
        types[i] = code(t);
        TYPE(types[i] >= 0, who, ": a tensor of type ", name_of(t), "; supported are float32, bfloat16 and float16");
        sizes[i] = t.numel();
        if (out) {
            const Tensor& o = (*out)[i];
            usable(who, o);
            VALUE(o.device() == t.device(), who, ": tensors on ", t.device(), " and ", o.device());
            VALUE(o.scalar_type() == t.scalar_type() && o.sizes() == t.sizes(), who, ": out must hold one tensor of the same type and shape per gradient");
            VALUE(o.is_contiguous() && !lazy(o), who, ": out must be contiguous");
            to[i] = sizes[i] ? o.data_ptr() : nullptr;
        }
        VALUE(out || !max_norm || !t._is_zerotensor(), who, ": a tensor without memory cannot be scaled in place");
        VALUE(out || !max_norm || sizes[i] == 0 || at::has_internal_overlap(t) != at::MemOverlap::Yes, who, ": a tensor whose elements share memory (an expanded one) cannot be scaled in place");
        // (in place a negative's memory is scaled like any other)
        if (t.is_contiguous() && !t._is_zerotensor() && !(out && t.is_neg())) from[i] = sizes[i] ? t.data_ptr() : nullptr;
        else {
            hold.push_back(whole(t));
            from[i] = hold.back().data_ptr();
            if (!out) back.push_back(i);
        }
        if (!out) to[i] = const_cast<void*>(from[i]);
    }
    if (max_norm) {
        // what is written may lie on nothing else, except that an output may be its own gradient
        struct Run { const char *lo, *hi; size_t i; bool in; };
        std::vector<Run> runs;
        runs.reserve(2 * n);
        for (size_t i = 0; i < n; ++i) {
            if (!sizes[i]) continue;
            // (a gradient with holes in it is read before anything is written, and may lie between another's elements: only its first one counts)
            const int64_t bytes = (out || src[i].is_non_overlapping_and_dense() ? sizes[i] : 1) * (types[i] == CCSP_OPS_F32 ? 4 : 2);
            const char* const w = (const char*)(out ? to[i] : src[i].data_ptr());
            runs.push_back({w, w + bytes, i, false});
            if (out && from[i] != to[i]) runs.push_back({(const char*)from[i], (const char*)from[i] + bytes, i, true});
        }
        std::sort(runs.begin(), runs.end(), [](const Run& a, const Run& b) { return a.lo < b.lo; });
        const char *end = nullptr, *end_written = nullptr;       // of everything, of what is written, up to here
        for (const Run& r : runs) {
            VALUE(r.lo >= (r.in ? end_written : end), who, ": a tensor to write appears twice or lies on another tensor");
            end = std::max(end, r.hi);
            if (!r.in) end_written = std::max(end_written, r.hi);
        }
    }
    const int64_t need = ccsp_ops_norm_workspace((int32_t)n, sizes.data());
    const Tensor res = at::empty({2}, src[0].options().dtype(at::kFloat)), ws = at::empty({need}, src[0].options().dtype(at::kByte));
    float* const r = res.data_ptr<float>();
    run(ccsp_ops_clip_norm((int32_t)n, from.data(), max_norm ? to.data() : nullptr, sizes.data(), types.data(), max_norm.value_or(0.0), r, r + 1, ptr(ws), need, on.stream));
    if (max_norm) {
        for (size_t i = 0; i < back.size(); ++i) src[back[i]].copy_(hold[i]);
        for (const Tensor& t : out ? *out : src)
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
    return res[0];
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const OpsError& e) {
            PyErr_SetString(g_ccsp_error ? g_ccsp_error : PyExc_RuntimeError, e.what());
        }
    });
    m.def("set_error", [](py::object e) { Py_XDECREF(g_ccsp_error); g_ccsp_error = e.release().ptr(); });
    m.def("version", [] { return ccsp_ops_version(); });
    py::class_<Plan, std::shared_ptr<Plan>>(m, "ExpertPlan", R"(What route() leaves on the device; all int32, made without waiting for the GPU.

offsets [E + 1]   first row of every expert; offsets[E] = active rows
rows [A]          row of every assignment, -1 if dropped
assign [A]        assignment of every row; behind the last active row ~a of the dropped ones
row_token [A]     token of every row, -1 behind the last active row
token_ptr [N + 1], token_assign [A]   with listed tokens: the active assignments of every token, ascending; else None
counts [E]        rows of every expert
shape             shape of the expert ids: the shape of combine_rows' weights)")
        .def_readonly("n_experts", &Plan::n_experts)
        .def_readonly("n_tokens", &Plan::n_tokens)
        .def_readonly("n_rows", &Plan::n_rows)
        .def_property_readonly("shape", [](const Plan& q) { return py::tuple(py::cast(q.shape)); })
        .def_property_readonly("device", [](const Plan& q) { return q.buf.device(); })
        .def_property_readonly("offsets", &Plan::offsets)
        .def_property_readonly("rows", &Plan::rows)
        .def_property_readonly("assign", &Plan::assign)
        .def_property_readonly("row_token", &Plan::row_token)
        .def_property_readonly("token_ptr", &Plan::token_ptr)
        .def_property_readonly("token_assign", &Plan::token_assign)
        .def_property_readonly("counts", &Plan::counts);
    m.def("route", &route);
    m.def("sort_rows", &sort_rows);
    m.def("combine_rows", &combine_rows);
    m.def("expert_linear", &expert_linear);
    m.def("clip", &clip);
}
