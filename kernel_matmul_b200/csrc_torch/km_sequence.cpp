// The sequence operators: argument checks, views, allocation and autograd for km_rotary, km_decay_attention,
// km_decay_gradient, km_decay_step and km_global_norm.
#include <ATen/MemoryOverlap.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <cmath>
#include <numeric>

#include "km_host.h"

namespace kmh {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

static int32_t type_of(const Tensor &t, const char *name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    switch (t.scalar_type()) {
        case at::kFloat: return KM_TYPE_F32;
        case at::kBFloat16: return KM_TYPE_BF16;
        case at::kHalf: return KM_TYPE_F16;
        default: TORCH_CHECK(false, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
    }
}

static void check_same_device(const Tensor &a, const Tensor &b) {
    TORCH_CHECK(a.device() == b.device(), "all tensors must be on the same CUDA device");
}

static void *stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// Whether a call has to go through its autograd function: for a gradient, or, so that it is refused there,
// for a forward-mode tangent.
static bool recording(std::initializer_list<const Tensor *> inputs) {
    for (const Tensor *t : inputs)
        if (t->defined() && ((t->requires_grad() && at::GradMode::is_enabled()) || t->_fw_grad(0).defined())) return true;
    return false;
}

// torch.jit.trace and make_fx see the allocation of a result and not the kernel that fills it: what they recorded would return
// memory as it comes.
static void refuse_recordings(const char *name) {
    // (both include keys in this thread's set; asking them costs a quarter of a microsecond)
    constexpr c10::DispatchKeySet keys({c10::DispatchKey::Tracer, c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot});
    if (!c10::impl::tls_local_dispatch_key_set().included_.has_any(keys)) return;
    TORCH_CHECK(!torch::jit::tracer::isTracing() &&
                    !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
                name, " cannot be recorded by torch.jit.trace or make_fx");
}

// In-place writes past autograd's back are counted, so that a graph that saved the tensor notices.
static void written(const Tensor &t) {
    if (!t.is_inference()) torch::autograd::increment_version(t);
}

// ------------------------------------------------------------------------------------------ rotary

struct RotaryCall {
    Tensor positions, frequencies;
    bool interleaved, inverse;
    double scale;
};

// xs: one or two tensors (batch.., tokens, heads, dim)
static std::vector<Tensor> rotary_raw(const std::vector<Tensor> &xs, const RotaryCall &c) {
    const Tensor &q = xs[0];
    const c10::cuda::CUDAGuard guard(q.device());
    const int64_t tokens = q.size(-3), dim = q.size(-1), lead = q.dim() - 3;
    std::vector<Tensor> in, out, result;
    km_view vin[2] = {}, vout[2] = {};
    int64_t heads[2] = {0, 0}, batch = 1;
    for (int64_t d = 0; d < lead; d++) batch *= q.size(d);
    for (size_t i = 0; i < xs.size(); i++) {
        result.push_back(at::empty(xs[i].sizes(), xs[i].options().requires_grad(false)));
        in.push_back(xs[i].reshape({batch, tokens, xs[i].size(-2), dim}));
        out.push_back(result[i].view({batch, tokens, xs[i].size(-2), dim}));
        heads[i] = xs[i].size(-2);
        for (auto [view, t] : {std::pair<km_view *, const Tensor *>{&vin[i], &in[i]}, {&vout[i], &out[i]}}) {
            view->data = t->data_ptr();
            view->batch_stride[0] = t->size(0) == 1 ? 0 : t->stride(0);
            view->batch_stride[1] = t->size(2) == 1 ? 0 : t->stride(2);
            view->stride[0] = t->size(1) == 1 ? 0 : t->stride(1);
            view->stride[1] = t->size(3) == 1 ? 1 : t->stride(3);
        }
    }
    Shape shape(q.sizes().begin(), q.sizes().end() - 2);
    Tensor p = c.positions;
    km_view vp{};
    if (p.dim() > 1) {
        p = p.expand(shape).reshape({batch, tokens});
        vp.batch_stride[0] = p.stride(0);
    }
    vp.data = p.data_ptr();
    vp.stride[0] = p.size(-1) == 1 ? 0 : p.stride(-1);
    const Tensor f = c.frequencies.contiguous();
    const int32_t ptype = p.scalar_type() == at::kInt ? KM_TYPE_I32 : p.scalar_type() == at::kLong ? KM_TYPE_I64 : KM_TYPE_F32;
    raise_on(km_rotary(type_of(q, "q"), batch, tokens, heads, dim, f.size(0), vin, vout, ptype, &vp,
                       f.scalar_type() == at::kDouble ? KM_TYPE_F64 : KM_TYPE_F32, f.data_ptr(), c.interleaved, c.inverse, (float)c.scale,
                       stream_of(q)));
    return result;
}

// Its gradient is the same rotation backwards, and so on.
struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
    static variable_list forward(AutogradContext *ctx, at::TensorList xs, const Tensor &positions, const Tensor &frequencies,
                                 bool interleaved, bool inverse, double scale) {
        ctx->save_for_backward({positions, frequencies});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["inverse"] = inverse;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["count"] = (int64_t)xs.size();
        return rotary_raw(xs.vec(), {positions, frequencies, interleaved, inverse, scale});
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const int64_t count = ctx->saved_data["count"].toInt();
        variable_list out((size_t)count + 5);
        std::vector<Tensor> given;
        std::vector<int64_t> which;
        for (int64_t i = 0; i < count; i++)
            if (grads[i].defined() && ctx->needs_input_grad(i)) given.push_back(grads[i]), which.push_back(i);
        if (given.empty()) return out;
        const bool interleaved = ctx->saved_data["interleaved"].toBool(), inverse = !ctx->saved_data["inverse"].toBool();
        const double scale = ctx->saved_data["scale"].toDouble();
        std::vector<Tensor> back;
        if (at::GradMode::is_enabled())  // (create_graph: the gradient itself is differentiable)
            back = RotaryFunction::apply(at::TensorList(given), s[0], s[1], interleaved, inverse, scale);
        else
            back = rotary_raw(given, {s[0], s[1], interleaved, inverse, scale});
        for (size_t j = 0; j < which.size(); j++) out[which[j]] = back[j];
        return out;
    }
};

std::vector<Tensor> rotary(const Tensor &q, const Maybe &k, const Tensor &positions, const Tensor &frequencies, bool interleaved,
                           double scale) {
    refuse_recordings("rotary");
    std::vector<Tensor> xs{q};
    if (k.has_value()) xs.push_back(*k);
    type_of(q, "q");
    TORCH_CHECK(q.dim() >= 3, "q must have the shape (batch.., tokens, heads, dim), got ", q.sizes());
    if (k.has_value()) {
        type_of(*k, "k");
        check_same_device(q, *k);
        TORCH_CHECK(k->scalar_type() == q.scalar_type(), "q and k must have the same type");
        TORCH_CHECK(k->dim() == q.dim() && k->sizes().slice(0, q.dim() - 2) == q.sizes().slice(0, q.dim() - 2) && k->size(-1) == q.size(-1),
                    "q and k must have the same batch, tokens and head size, got ", q.sizes(), " and ", k->sizes());
    }
    check_same_device(q, positions), check_same_device(q, frequencies);
    const auto pt = positions.scalar_type();
    TORCH_CHECK(pt == at::kInt || pt == at::kLong || pt == at::kFloat, "positions must be int32, int64 or float32");
    TORCH_CHECK(frequencies.scalar_type() == at::kFloat || frequencies.scalar_type() == at::kDouble, "frequencies must be float32 or float64");
    TORCH_CHECK(frequencies.dim() == 1, "frequencies must have one dim");
    TORCH_CHECK(2 * frequencies.size(0) <= q.size(-1), "frequencies for ", 2 * frequencies.size(0), " values of a head of ", q.size(-1));
    TORCH_CHECK(positions.dim() >= 1 && positions.dim() <= q.dim() - 2 && positions.size(-1) == q.size(-3),
                "positions must have the shape (tokens,) or (batch.., tokens), got ", positions.sizes(), " for q ", q.sizes());
    const int64_t shift = q.dim() - 2 - positions.dim();
    for (int64_t d = 0; d + 1 < positions.dim(); d++)
        TORCH_CHECK(positions.size(d) == q.size(d + shift) || positions.size(d) == 1, "positions ", positions.sizes(),
                    " do not broadcast to the tokens of q ", q.sizes());
    TORCH_CHECK(!positions.requires_grad() && !frequencies.requires_grad(), "rotary has no gradient for positions or frequencies");
    if (recording({&xs[0], &xs.back()}))
        return RotaryFunction::apply(at::TensorList(xs), positions, frequencies, interleaved, false, scale);
    return rotary_raw(xs, {positions, frequencies, interleaved, false, scale});
}

// ------------------------------------------------------------------------------------------ linear attention with decay

// One call's operands as 4-d tensors (sequence, token, head, value), states (sequence, head, dk, dv).
struct DecayCall {
    Tensor q, k, v, log_decay, initial, starts;  // initial, starts: undefined if absent
    int64_t sequences, tokens, heads, groups, dk, dv;
    double scale;
    int64_t path;
    int32_t type;

    km_decay_problem problem(int32_t reverse, bool transposed, bool wide) const {
        km_decay_problem p{};
        p.dtype = type, p.out_dtype = wide ? KM_TYPE_F32 : type;
        p.reverse = reverse, p.path = (int32_t)path;
        p.sequences = sequences, p.tokens = tokens, p.groups = groups, p.group = heads / groups;
        p.dk = transposed ? dv : dk, p.dv = transposed ? dk : dv;
        p.packed = starts.defined();
        p.scale = (float)scale;
        return p;
    }
    // An operand of the tensor-core kernels, which load rows that start on boundaries of 16 bytes by TMA and any others value by
    // value: those are copied into such rows first, but for sequences of a few tokens (4 heads of 33 and 77: 500 tokens take
    // 159 us without the copies and 49 with them, 64 tokens 46 and 45; a token's three copies cost 10 us of host time).
    Tensor ready(const Tensor &t) const {
        if (type == KM_TYPE_F32 || path == PATH_FMA || t.size(1) < 16) return t;
        bool aligned = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
        for (int64_t d = 0; d < 3; d++) aligned = aligned && (t.size(d) == 1 || (t.stride(d) % 8 == 0 && (d != 1 || t.stride(d) > 0)));
        if (aligned) return t;
        at::NoGradGuard no_grad;
        const Tensor rows = at::empty({t.size(0), t.size(1), t.size(2), (t.size(3) + 7) / 8 * 8}, t.options().requires_grad(false)).narrow(3, 0, t.size(3));
        return rows.copy_(t);
    }
    // (sequence, token, head, value) with all heads, or one for each group
    km_view tokens_view(const Tensor &t) const {
        km_view v{};
        const int64_t group = heads / groups;
        v.data = t.data_ptr();
        v.batch_stride[0] = t.size(0) == 1 ? 0 : t.stride(0);
        const bool shared = t.size(2) == groups;
        v.batch_stride[1] = shared ? t.stride(2) : t.stride(2) * group;
        v.batch_stride[2] = shared ? 0 : t.stride(2);
        if (t.size(2) == 1) v.batch_stride[1] = 0;
        v.stride[0] = t.stride(1);
        v.stride[1] = t.size(3) == 1 ? 1 : t.stride(3);
        return v;
    }
    km_view state_view(const Tensor &t, bool transposed) const {
        km_view v{};
        if (!t.defined()) return v;
        v.data = t.data_ptr();
        v.batch_stride[0] = t.stride(0);
        v.batch_stride[1] = t.stride(1) * (heads / groups);
        v.batch_stride[2] = t.stride(1);
        v.stride[0] = t.stride(transposed ? 3 : 2);
        v.stride[1] = t.stride(transposed ? 2 : 3);
        return v;
    }
    const int32_t *starts_ptr() const { return starts.defined() ? starts.const_data_ptr<int32_t>() : nullptr; }

    // `states`: the workspace of a call over the same states with dk and dv swapped (undefined: none).  Returns this call's own.
    Tensor run(int32_t reverse, bool transposed, const Tensor &ta, const Tensor &tb, const Tensor &tc, const Tensor &out, const Tensor &state_in,
               const Tensor &state_out, const Tensor &states = Tensor()) const {
        const Tensor a = ready(ta), b = ready(tb), c = ready(tc);
        km_decay_problem p = problem(reverse, transposed, out.scalar_type() == at::kFloat);
        if (sequences == 0) {  // (no launch will write the rows of no sequence)
            out.zero_();
            return Tensor();
        }
        const km_view va = tokens_view(a), vb = tokens_view(b), vc = tokens_view(c), vo = tokens_view(out),
                      vi = state_view(state_in, transposed), vs = state_view(state_out, transposed);
        const size_t bytes = km_decay_attention_workspace_bytes(&p);
        p.states = bytes && states.defined() ? 2 : 0;
        const Tensor ws = !bytes ? Tensor() : p.states ? states : workspace(q, bytes);
        raise_on(km_decay_attention(&p, &va, &vb, &vc, &vo, log_decay.const_data_ptr<float>(), starts_ptr(), &vi, &vs,
                                    bytes ? ws.data_ptr() : nullptr, bytes, stream_of(q)));
        return ws;
    }
    Tensor state_like() const { return at::empty({sequences, heads, dk, dv}, q.options().dtype(at::kFloat).requires_grad(false)); }
    Tensor result_like() const { return at::empty({q.size(0), tokens, heads, dv}, q.options().requires_grad(false)); }
    // per-head results of `dim` values summed over the heads of a group
    Tensor summed(bool transposed, const Tensor &a, const Tensor &b, const Tensor &c, int64_t dim, const Tensor &state_in,
                  const Tensor &state_out, Tensor &states) const {
        const auto opt = q.options().requires_grad(false);
        const int64_t group = heads / groups;
        Tensor out = at::empty({q.size(0), tokens, heads, dim}, group > 1 ? opt.dtype(at::kFloat) : opt);
        states = run(1, transposed, a, b, c, out, state_in, state_out, states);
        if (group == 1) return out;
        Tensor sums = at::empty({q.size(0), tokens, groups, dim}, opt);
        raise_on(km_group_sums(type, q.size(0) * tokens, groups, group, dim, out.const_data_ptr<float>(), sums.data_ptr(), stream_of(q)));
        return sums;
    }
};

static variable_list decay_forward(const DecayCall &c, bool return_state, Tensor *states = nullptr) {
    const c10::cuda::CUDAGuard guard(c.q.device());
    poll_gave_up(c.q.device().index());
    Tensor out = c.result_like(), state = return_state ? c.state_like() : Tensor();
    const Tensor ws = c.run(0, false, c.q, c.k, c.v, out, c.initial, state);
    if (states != nullptr) *states = ws;
    return return_state ? variable_list{out, state} : variable_list{out};
}

struct DecayFunction : torch::autograd::Function<DecayFunction> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay,
                                 const Maybe &initial, const Maybe &starts, const DecayCall &call, bool return_state) {
        DecayCall c = call;  // (the inputs as the function sees them)
        c.q = c.ready(q), c.k = c.ready(k), c.v = c.ready(v), c.log_decay = log_decay, c.initial = initial.value_or(Tensor()), c.starts = starts.value_or(Tensor());
        Tensor states;  // between segments, for the gradient of q
        variable_list out = decay_forward(c, return_state, &states);
        ctx->save_for_backward({c.q, c.k, c.v, log_decay, c.initial, c.starts, states});
        ctx->saved_data["sizes"] = std::vector<int64_t>{c.sequences, c.tokens, c.heads, c.groups, c.dk, c.dv, c.path, c.type};
        ctx->saved_data["scale"] = c.scale;
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "decay_attention has no second derivative (create_graph)");
        const auto s = ctx->get_saved_variables();
        const auto n = ctx->saved_data["sizes"].toIntVector();
        const DecayCall c{s[0], s[1], s[2], s[3], s[4], s[5], n[0], n[1], n[2], n[3], n[4], n[5], ctx->saved_data["scale"].toDouble(), n[6], (int32_t)n[7]};
        variable_list out(8);
        const Tensor ds = grads.size() > 1 ? grads[1] : Tensor();
        Tensor go = grads[0];
        if (!go.defined() && !ds.defined()) return out;
        const c10::cuda::CUDAGuard guard(c.q.device());
        poll_gave_up(c.q.device().index());
        if (!go.defined()) go = at::zeros({1}, c.q.options().requires_grad(false)).expand({c.q.size(0), c.tokens, c.heads, c.dv});
        go = c.ready(go);
        if (ctx->needs_input_grad(0)) {
            out[0] = at::empty({c.q.size(0), c.tokens, c.heads, c.dk}, c.q.options().requires_grad(false));
            c.run(2, true, go, c.v, c.k, out[0], c.initial, Tensor(), s[6]);
        }
        const bool initial = c.initial.defined() && ctx->needs_input_grad(4);
        Tensor back;  // the states of the way back, which the gradients of v and k share
        if (ctx->needs_input_grad(2) || initial) {
            if (initial) out[4] = c.state_like();
            out[2] = c.summed(false, c.k, c.q, go, c.dv, ds, out[4], back);
        }
        if (ctx->needs_input_grad(1)) out[1] = c.summed(true, c.v, go, c.q, c.dk, ds, Tensor(), back);
        if (ctx->needs_input_grad(3)) {
            const km_decay_problem p = c.problem(0, false, false);
            out[3] = at::empty({c.heads}, c.log_decay.options().requires_grad(false));
            const size_t bytes = km_decay_gradient_workspace_bytes(&p);
            const Tensor ws = workspace(c.q, bytes);
            const km_view vq = c.tokens_view(c.q), vk = c.tokens_view(c.k), vv = c.tokens_view(c.v), vd = c.tokens_view(go),
                          vi = c.state_view(c.initial, false), vs = c.state_view(ds, false);
            raise_on(km_decay_gradient(&p, &vq, &vk, &vv, &vd, c.log_decay.const_data_ptr<float>(), c.starts_ptr(), &vi, &vs,
                                       out[3].data_ptr<float>(), ws.data_ptr(), (size_t)ws.numel(), stream_of(c.q)));
        }
        return out;
    }
};

static double scale_for(std::optional<double> scale, int64_t dk) { return scale.value_or(1.0 / std::sqrt((double)std::max<int64_t>(dk, 1))); }

std::vector<Tensor> decay_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay, std::optional<double> scale,
                                    const Maybe &initial_state, const Maybe &starts, bool return_state, int64_t path) {
    refuse_recordings("decay_attention");
    DecayCall c{};
    c.type = type_of(q, "q");
    type_of(k, "k"), type_of(v, "v"), check_f32(log_decay);
    check_same_device(q, k), check_same_device(q, v), check_same_device(q, log_decay);
    TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "q, k and v must have the same type");
    TORCH_CHECK(path != PATH_TC || c.type != KM_TYPE_F32, "path 'tc' takes bfloat16 and float16 operands");
    if (path != PATH_AUTO && path != PATH_FMA && path != PATH_TC) throw ArgumentError("path must be 'auto', 'fma' or 'tc'");
    const bool packed = starts.has_value();
    TORCH_CHECK(q.dim() >= 3 && (!packed || q.dim() == 3), "q must have the shape ", packed ? "(tokens, heads, dk) with sequence_starts" : "(batch.., tokens, heads, dk)",
                ", got ", q.sizes());
    const int64_t lead = q.dim() - 3;
    TORCH_CHECK(k.dim() == q.dim() && v.dim() == q.dim() && k.sizes().slice(0, lead + 1) == q.sizes().slice(0, lead + 1) &&
                    v.sizes().slice(0, lead + 2) == k.sizes().slice(0, lead + 2) && k.size(-1) == q.size(-1),
                "k (batch.., tokens, groups, dk) and v (batch.., tokens, groups, dv) must agree with q ", q.sizes(), ", got ", k.sizes(), " and ", v.sizes());
    c.tokens = q.size(-3), c.heads = q.size(-2), c.groups = k.size(-2), c.dk = q.size(-1), c.dv = v.size(-1);
    TORCH_CHECK(c.groups > 0 ? c.heads % c.groups == 0 && c.heads > 0 : c.heads == 0, "the heads of q (", c.heads, ") must be a multiple of those of k and v (", c.groups, ")");
    TORCH_CHECK(c.dk >= 1 && c.dk <= KM_DECAY_MAX_DIM && c.dv >= 1 && c.dv <= KM_DECAY_MAX_DIM, "head sizes must be 1 to ", KM_DECAY_MAX_DIM,
                ", got ", c.dk, " and ", c.dv);
    TORCH_CHECK(log_decay.dim() == 1 && log_decay.size(0) == c.heads, "log_decay must have the shape (heads,) = (", c.heads, ",), got ", log_decay.sizes());
    c.scale = scale_for(scale, c.dk), c.path = path;
    Shape batch(q.sizes().begin(), q.sizes().begin() + lead), state_shape(batch);
    int64_t count = 1;
    for (int64_t b : batch) count *= b;
    c.sequences = count;
    if (packed) {
        check_i32(*starts);
        check_same_device(q, *starts);
        TORCH_CHECK(starts->dim() == 1 && starts->size(0) >= 1, "sequence_starts must have the shape (sequences + 1,), got ", starts->sizes());
        c.sequences = starts->size(0) - 1;
        state_shape = {c.sequences};
        c.starts = starts->contiguous();
    }
    state_shape.insert(state_shape.end(), {c.heads, c.dk, c.dv});
    if (initial_state.has_value()) {
        check_f32(*initial_state);
        check_same_device(q, *initial_state);
        TORCH_CHECK(initial_state->sizes() == at::IntArrayRef(state_shape), "initial_state must have the shape ", at::IntArrayRef(state_shape), ", got ", initial_state->sizes());
    }
    // (views where the batch dims collapse; differentiable either way)
    c.q = q.reshape({count, c.tokens, c.heads, c.dk});
    c.k = k.reshape({count, c.tokens, c.groups, c.dk});
    c.v = v.reshape({count, c.tokens, c.groups, c.dv});
    c.log_decay = log_decay.contiguous();
    if (initial_state.has_value()) c.initial = initial_state->reshape({c.sequences, c.heads, c.dk, c.dv});
    variable_list r;
    if (c.heads == 0) {  // nothing to launch for, nothing to differentiate
        r = {at::empty({count, c.tokens, 0, c.dv}, q.options().requires_grad(false))};
        if (return_state) r.push_back(c.state_like());
    } else if (recording({&c.q, &c.k, &c.v, &c.log_decay, &c.initial})) {
        const auto maybe = [](const Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); };
        r = DecayFunction::apply(c.q, c.k, c.v, c.log_decay, maybe(c.initial), maybe(c.starts), c, return_state);
    } else {
        r = decay_forward(c, return_state);
    }
    Shape shape(batch);
    shape.insert(shape.end(), {c.tokens, c.heads, c.dv});
    r[0] = r[0].view(shape);
    if (return_state) r[1] = r[1].view(state_shape);
    return r;
}

Tensor decay_attention_step(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay, const Tensor &states,
                            std::optional<double> scale, const Maybe &slots) {
    refuse_recordings("decay_attention_step");
    const int32_t type = type_of(q, "q");
    type_of(k, "k"), type_of(v, "v"), check_f32(log_decay), check_f32(states);
    check_same_device(q, k), check_same_device(q, v), check_same_device(q, log_decay), check_same_device(q, states);
    TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "q, k and v must have the same type");
    TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3 && k.size(0) == q.size(0) && v.size(0) == q.size(0) && k.size(2) == q.size(2) &&
                    v.size(1) == k.size(1),
                "q (rows, heads, dk), k (rows, groups, dk) and v (rows, groups, dv) must agree, got ", q.sizes(), ", ", k.sizes(), " and ", v.sizes());
    const int64_t rows = q.size(0), heads = q.size(1), groups = k.size(1), dk = q.size(2), dv = v.size(2);
    TORCH_CHECK(groups > 0 ? heads % groups == 0 && heads > 0 : heads == 0, "the heads of q (", heads, ") must be a multiple of those of k and v (", groups, ")");
    TORCH_CHECK(dk >= 1 && dk <= KM_DECAY_MAX_DIM && dv >= 1 && dv <= KM_DECAY_MAX_DIM, "head sizes must be 1 to ", KM_DECAY_MAX_DIM, ", got ", dk,
                " and ", dv);
    TORCH_CHECK(log_decay.dim() == 1 && log_decay.size(0) == heads, "log_decay must have the shape (heads,) = (", heads, ",), got ", log_decay.sizes());
    TORCH_CHECK(states.dim() == 4 && states.size(1) == heads && states.size(2) == dk && states.size(3) == dv,
                "states must have the shape (slots, heads, dk, dv), got ", states.sizes());
    TORCH_CHECK(dv == 1 || states.stride(3) == 1, "the last dim of states must be contiguous");
    at::assert_no_internal_overlap(states);
    TORCH_CHECK(!recording({&q, &k, &v, &log_decay, &states}), "decay_attention_step updates states in place and has no gradient: use decay_attention");
    Tensor sl;
    int32_t slot_type = KM_TYPE_I32;
    if (slots.has_value()) {
        check_same_device(q, *slots);
        TORCH_CHECK(slots->scalar_type() == at::kInt || slots->scalar_type() == at::kLong, "slots must be int32 or int64");
        TORCH_CHECK(slots->dim() == 1 && slots->size(0) == rows, "slots must have the shape (rows,) = (", rows, ",), got ", slots->sizes());
        sl = slots->contiguous();
        slot_type = sl.scalar_type() == at::kInt ? KM_TYPE_I32 : KM_TYPE_I64;
    } else {
        TORCH_CHECK(states.size(0) == rows, "without slots there must be one state for each row, got ", states.size(0), " for ", rows);
    }
    const c10::cuda::CUDAGuard guard(q.device());
    Tensor out = at::empty({rows, heads, dv}, q.options().requires_grad(false));
    if (rows == 0 || heads == 0) return out;
    const int64_t group = heads / groups;
    std::vector<Tensor> keep;
    const auto rows_view = [&](const Tensor &t) {
        keep.push_back(t.size(2) == 1 || t.stride(2) == 1 ? t : t.contiguous());
        const Tensor &x = keep.back();
        km_view r{};
        const bool shared = x.size(1) == groups;
        r.data = x.data_ptr();
        r.batch_stride[0] = x.stride(0);
        r.batch_stride[1] = shared ? x.stride(1) : x.stride(1) * group;
        r.batch_stride[2] = shared ? 0 : x.stride(1);
        r.stride[1] = 1;
        return r;
    };
    const km_view vq = rows_view(q), vk = rows_view(k), vv = rows_view(v), vo = rows_view(out);
    km_view vs{};
    vs.data = states.data_ptr();
    vs.batch_stride[0] = states.stride(0), vs.batch_stride[1] = states.stride(1) * group, vs.batch_stride[2] = states.stride(1);
    vs.stride[0] = states.stride(2), vs.stride[1] = 1;
    const Tensor g = log_decay.contiguous();
    raise_on(km_decay_step(type, rows, states.size(0), groups, group, dk, dv, &vq, &vk, &vv, &vo, g.const_data_ptr<float>(), &vs, slot_type,
                           sl.defined() ? sl.data_ptr() : nullptr, (float)scale_for(scale, dk), stream_of(q)));
    written(states);
    return out;
}

// ------------------------------------------------------------------------------------------ norm over many tensors

// Whether views `a` and `b` are shown to share no element.  With strides S_1 > S_2 > .. > 1 of both, an element at offset
// i_1 S_1 + i_2 S_2 + .. has these numbers as digits, and only these as long as no digit with all below it reaches the stride above.  A
// view's elements are a box in the digits; they are apart where the boxes are, in any one digit.
static bool apart_from(const Tensor &a, const Tensor &b, uintptr_t origin) {
    const int64_t size = a.itemsize();
    if (b.itemsize() != size) return false;
    std::vector<int64_t> strides{1};
    for (const Tensor *t : {&a, &b})
        for (int64_t d = 0; d < t->dim(); d++)
            if (t->size(d) > 1) strides.push_back(t->stride(d));
    std::sort(strides.begin(), strides.end(), std::greater<>());
    strides.erase(std::unique(strides.begin(), strides.end()), strides.end());
    if (strides.back() < 1) return false;
    const size_t n = strides.size();
    std::vector<int64_t> first[2], behind[2];
    for (int which = 0; which < 2; which++) {
        const Tensor &t = which ? b : a;
        const uintptr_t from = reinterpret_cast<uintptr_t>(t.data_ptr()) - origin;
        if (from % size != 0) return false;
        int64_t rest = (int64_t)(from / size);
        for (size_t i = 0; i < n; i++) {
            first[which].push_back(rest / strides[i]), rest %= strides[i];
            int64_t count = 1;
            for (int64_t d = 0; d < t.dim(); d++) {
                if (t.size(d) <= 1 || t.stride(d) != strides[i]) continue;
                if (count > 1) return false;  // (two dims of one stride)
                count = t.size(d);
            }
            behind[which].push_back(first[which][i] + count);
        }
    }
    bool apart = false;
    int64_t below = 0;  // the largest offset of the digits below
    for (size_t i = n; i-- > 0;) {
        if (below >= strides[i]) return false;
        if (i > 0) below += (std::max(behind[0][i], behind[1][i]) - 1) * strides[i];
        apart = apart || behind[0][i] <= first[1][i] || behind[1][i] <= first[0][i];
    }
    return apart;
}

// Seen from the start of their buffer, or from the first of them.
static bool apart(const Tensor &a, const Tensor &b) {
    const auto at = [](const Tensor &t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); };
    const auto buffer = [](const Tensor &t) { return reinterpret_cast<uintptr_t>(t.storage().data()); };
    return (buffer(a) == buffer(b) && apart_from(a, b, buffer(a))) || apart_from(a, b, std::min(at(a), at(b)));
}

static Tensor norm_raw(const std::vector<Tensor> &tensors, std::optional<double> max_norm, double eps) {
    const bool scale = max_norm.has_value();
    const size_t n = tensors.size();
    std::vector<Tensor> flat;  // dense storage to work on
    flat.reserve(n);
    for (const Tensor &t : tensors) {
        type_of(t, "x");
        check_same_device(tensors[0], t);
        TORCH_CHECK(t.layout() == at::kStrided, "tensors must be strided");
        if (scale) {
            TORCH_CHECK(!(t.requires_grad() && t.is_leaf()), "clip_global_norm_ takes gradients, not the parameters that require them");
            at::assert_no_internal_overlap(t);
        }
        flat.push_back(t.is_non_overlapping_and_dense() ? t : t.contiguous());
    }
    const c10::cuda::CUDAGuard guard(tensors[0].device());
    // a tensor that is listed twice counts once and is scaled once; tensors that overlap otherwise are not scaled at all
    std::vector<uintptr_t> begin(n), end(n, 0);
    for (size_t i = 0; i < n; i++) begin[i] = reinterpret_cast<uintptr_t>(tensors[i].data_ptr());
    std::vector<size_t> order(n);
    std::iota(order.begin(), order.end(), (size_t)0);
    std::stable_sort(order.begin(), order.end(), [&](size_t a, size_t b) { return begin[a] < begin[b]; });
    std::vector<char> repeated(n, 0);
    std::vector<size_t> open;  // earlier tensors that reach behind this one's first element
    for (size_t i : order) {
        const Tensor &t = tensors[i];
        if (t.numel() == 0) continue;
        // (the extent of a view with gaps)
        uintptr_t span = 1;
        for (int64_t d = 0; d < t.dim(); d++) span += (uintptr_t)((t.size(d) - 1) * t.stride(d));
        end[i] = begin[i] + span * t.itemsize();
        open.erase(std::remove_if(open.begin(), open.end(), [&](size_t j) { return end[j] <= begin[i]; }), open.end());
        for (size_t j : open)
            repeated[i] = repeated[i] || (begin[i] == begin[j] && t.sizes() == tensors[j].sizes() && t.strides() == tensors[j].strides() &&
                                          t.scalar_type() == tensors[j].scalar_type());
        if (repeated[i]) continue;
        if (scale)
            for (size_t j : open) TORCH_CHECK(apart(tensors[j], t), "tensors to clip must not overlap");
        open.push_back(i);
    }
    std::vector<void *> data;
    std::vector<int64_t> elements;
    std::vector<int32_t> types;
    for (size_t i = 0; i < n; i++) {
        if (repeated[i]) continue;
        data.push_back(flat[i].data_ptr()), elements.push_back(flat[i].numel()), types.push_back(type_of(flat[i], "x"));
    }
    Tensor norm = at::empty({}, tensors[0].options().dtype(at::kFloat).requires_grad(false));
    const Tensor ws = workspace(norm, km_global_norm_workspace_bytes((int64_t)data.size()));
    raise_on(km_global_norm((int64_t)data.size(), data.data(), elements.data(), types.data(), scale, max_norm.value_or(0.0), eps,
                            norm.data_ptr<float>(), ws.data_ptr(), (size_t)ws.numel(), stream_of(norm)));
    if (scale) {
        for (size_t i = 0; i < n; i++) {
            if (repeated[i]) continue;
            if (flat[i].is_same(tensors[i])) {
                written(tensors[i]);
            } else {
                at::NoGradGuard no_grad;
                tensors[i].copy_(flat[i]);
            }
        }
    }
    return norm;
}

// A norm of tensors that require a gradient says that it has none where one is asked for, instead of leaving it out of a sum.
struct NormFunction : torch::autograd::Function<NormFunction> {
    static Tensor forward(AutogradContext *, at::TensorList tensors) { return norm_raw(tensors.vec(), {}, 0.0); }
    static variable_list backward(AutogradContext *, variable_list) { TORCH_CHECK(false, "global_norm has no gradient"); }
};

Tensor global_norm(const std::vector<Tensor> &tensors, std::optional<double> max_norm, double eps) {
    refuse_recordings("global_norm");
    if (tensors.empty()) throw ArgumentError("no tensors given");
    if (max_norm.has_value() && !(*max_norm >= 0.0)) throw ArgumentError("max_norm must not be negative or NaN");
    if (!(eps >= 0.0) || std::isinf(eps)) throw ArgumentError("eps must be finite and not negative");
    if (!max_norm.has_value()) {
        for (const Tensor &t : tensors)
            if (recording({&t})) return NormFunction::apply(at::TensorList(tensors));
    } else if (torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr) {  // (the question of each tensor takes a lock)
        for (const Tensor &t : tensors) TORCH_CHECK(!t._fw_grad(0).defined(), "clip_global_norm_ has no forward-mode derivative");
    }
    return norm_raw(tensors, max_norm, eps);
}

}  // namespace kmh
