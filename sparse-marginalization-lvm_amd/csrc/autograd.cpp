// The autograd nodes of the layers, the log-probabilities and the policy loss, and the optimiser's table, over the
// C ABI of include/sparsemarg.h.  Host side only: output allocation, what is kept for the backward, the calls.
//
// In C++ because these operators train small models, where a step is host time.  The engine runs a node's
// backward on a thread of its own, and a node written in Python has to hand the interpreter's lock over twice
// for it (an empty one costs 59 us, forward and backward, where the kernels of a small layer take 10).
// Arguments of the nodes are checked by their callers, lvmhelpers/functional.py.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "../../include/sparsemarg.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

int32_t kind_of(at::ScalarType type)
{
    switch (type) {
        case at::kFloat: return SMLVM_F32;
        case at::kHalf: return SMLVM_F16;
        case at::kBFloat16: return SMLVM_BF16;
        default: TORCH_CHECK_TYPE(false, "expected float32, float16 or bfloat16, got ", type);
    }
}
int32_t kind_of(const Tensor& t) { return kind_of(t.scalar_type()); }

struct NativeError : std::runtime_error { using std::runtime_error::runtime_error; };   // lvmhelpers._native.NativeError

void check(int rc, const char* what)
{
    if (rc != SMLVM_OK)
        throw NativeError(c10::str(what, ": ", smlvm_error_string(rc), " (code ", rc, ", hip error ", smlvm_last_hip_error(), ")"));
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(const Maybe& t) { return t ? ptr(*t) : nullptr; }
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants(const Maybe& t) { return t && wants(*t); }

// Forward-mode derivatives: a dual tensor need not require a gradient, and its tangent would be lost without a word.
void no_tangent(const Tensor& t)
{
    if (t.defined() && t._fw_grad(/*level=*/0).defined())
        C10_THROW_ERROR(NotImplementedError, "this operator has no forward-mode derivative");
}
void no_tangent(const Maybe& t) { if (t) no_tangent(*t); }
template <class... Ts> void no_tangents(const Ts&... t) { (no_tangent(t), ...); }

Tensor workspace(size_t bytes, const Tensor& like)
{
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// Gradients that are differentiable no further: where a graph of the backward is recorded and could reach them,
// they hang on a node that says so.
struct Once : Function<Once> {
    static Tensor forward(AutogradContext*, const Tensor& grad, const at::TensorList&) { return grad.alias(); }
    static variable_list backward(AutogradContext*, const variable_list&)
    {
        TORCH_CHECK(false, "this operator's gradient cannot be differentiated again (once_differentiable)");
    }
};
void once(variable_list& grads, const variable_list& reached_from)
{
    if (!at::GradMode::is_enabled()) return;
    variable_list from;
    for (const Tensor& t : reached_from) if (wants(t)) from.push_back(t);
    if (from.empty()) return;
    for (Tensor& g : grads) if (g.defined()) g = Once::apply(g, at::TensorList(from));
}

// A matrix whose rows are consecutive elements, any distance apart.
struct Rows {
    Tensor t;
    int64_t ld;
    Rows(const Tensor& m) : t(m)
    {
        const int64_t width = m.size(1);
        if (!m.is_contiguous() && ((width > 1 && m.stride(1) != 1) || (m.size(0) > 1 && m.stride(0) < width))) t = m.contiguous();
        ld = t.is_contiguous() ? width : std::max(t.stride(0), width);
    }
};

enum { kRelu = 1 };

// relu's slope can be told from its result, but for fp16's: arguments below 2^-25 have the result 0 there.
bool sign_of_y(int64_t act, int32_t kind, bool residual) { return act == kRelu && !residual && kind != SMLVM_F16; }

Tensor linear_forward(const Tensor& x_, const Tensor& w_, const Maybe& b, const Maybe& r_, int64_t act, Tensor* pre)
{
    const c10::DeviceGuard guard(x_.device());
    const int64_t M = x_.size(0), K = x_.size(1), N = w_.size(0);
    const int32_t kind = kind_of(x_);
    const Rows x(x_), w(w_);
    std::optional<Rows> r;
    if (r_) r.emplace(*r_);
    Tensor y = at::empty({M, N}, x_.options());
    if (pre) *pre = at::empty({M, N}, x_.options().dtype(kind == SMLVM_F32 || (kind == SMLVM_F16 && act != kRelu) ? at::kFloat : at::kHalf));
    const size_t bytes = smlvm_linear_fwd_workspace_bytes(kind, M, N, K);
    const Tensor ws = workspace(bytes, x_);
    check(smlvm_linear_fwd(ptr(x.t), x.ld, ptr(w.t), w.ld, ptr(b), r ? ptr(r->t) : nullptr, r ? r->ld : N, ptr(y),
                           pre ? ptr(*pre) : nullptr, kind, (int32_t)act, M, N, K, ptr(ws), bytes, stream_of(x_)),
          "smlvm_linear_fwd");
    return y;
}

// act(x w^T + b) + r.  For the backward the forward leaves act's argument (include/sparsemarg.h says in which type), or
// relu's result in its place.
struct LinearAct : Function<LinearAct> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Maybe& b, const Maybe& r, int64_t act)
    {
        const bool need = wants(x) || wants(w) || wants(b), own_sign = sign_of_y(act, kind_of(x), r.has_value());
        Tensor pre;
        Tensor y = linear_forward(x, w, b, r, act, need && act && !own_sign ? &pre : nullptr);
        ctx->saved_data["act"] = act;
        ctx->saved_data["inputs"] = (int64_t)((b ? 1 : 0) | (r ? 2 : 0));
        if (need) ctx->save_for_backward(!act ? variable_list{x, w} : variable_list{x, w, own_sign ? y : pre});
        return y;
    }

    static variable_list backward(AutogradContext* ctx, const variable_list& grads)
    {
        const int64_t act = ctx->saved_data["act"].toInt(), inputs = ctx->saved_data["inputs"].toInt();
        const bool has_b = inputs & 1, has_r = inputs & 2;
        const bool want_dx = ctx->needs_input_grad(0), want_dw = ctx->needs_input_grad(1);
        const bool want_db = has_b && ctx->needs_input_grad(2), want_dr = has_r && ctx->needs_input_grad(has_b ? 3 : 2);
        Tensor dx, dw, db;
        if (want_dx || want_dw || want_db) {
            const variable_list saved = ctx->get_saved_variables();
            const Tensor& x_ = saved[0];
            const c10::DeviceGuard guard(x_.device());
            const int64_t M = x_.size(0), K = x_.size(1), N = saved[1].size(0);
            const int32_t kind = kind_of(x_);
            const Rows x(x_), w(saved[1]), dy(act ? grads[0].contiguous() : grads[0]);
            if (want_dx) dx = at::empty({M, K}, x_.options());
            if (want_dw || want_db) dw = at::empty({N, K}, x_.options());
            if (want_db) db = at::empty({N}, x_.options());
            const size_t bytes = smlvm_linear_bwd_workspace_bytes(kind, (int32_t)act, M, N, K);
            const Tensor ws = workspace(bytes, x_);
            check(smlvm_linear_bwd(ptr(dy.t), dy.ld, act ? ptr(saved[2]) : nullptr, sign_of_y(act, kind, has_r), ptr(x.t), x.ld, ptr(w.t),
                                   w.ld, ptr(dx), ptr(dw), ptr(db), kind, (int32_t)act, M, N, K, ptr(ws), bytes, stream_of(x_)),
                  "smlvm_linear_bwd");
            if (!want_dw) dw = Tensor();
            variable_list out = {dx, dw, db};
            once(out, {grads[0], x_, saved[1]});
            dx = out[0]; dw = out[1]; db = out[2];
        }
        return {dx, dw, db, want_dr ? grads[0] : Tensor(), Tensor()};
    }
};

Tensor linear_act(const Tensor& x, const Tensor& w, const Maybe& b, const Maybe& r, int64_t act)
{
    no_tangents(x, w, b, r);
    if (at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b) || wants(r))) return LinearAct::apply(x, w, b, r, act);
    return linear_forward(x, w, b, r, act, nullptr);
}

// logits [B, T, V], one row's elements consecutive (B and T in any stride)
Tensor rows_of(const Tensor& logits)
{
    return logits.size(2) > 1 && logits.stride(2) != 1 ? logits.contiguous() : logits;
}

// dlogits = g (c dlogp + h dentropy); ready: a buffer that holds the result for g = 1 already (it is written only
// where g is another number)
Tensor rows_backward(const Tensor& logits, const Tensor& actions, const Tensor& mask, const float* stats, const float* c, const float* h,
                     const Tensor& g, const Tensor& ready)
{
    const c10::DeviceGuard guard(logits.device());
    const Tensor z = rows_of(logits);
    Tensor out = ready.defined() ? ready : at::empty({z.size(0), z.size(1), z.size(2)}, z.options());
    check(smlvm_token_logprobs_bwd(ptr(z), kind_of(z), z.stride(0), z.stride(1), static_cast<const int64_t*>(ptr(actions)),
                                   static_cast<const uint8_t*>(ptr(mask)), stats, c, h, static_cast<const float*>(ptr(g)),
                                   ready.defined() ? 1 : 0, ptr(out), z.size(0), z.size(1), z.size(2), stream_of(z)),
          "smlvm_token_logprobs_bwd");
    return out;
}

variable_list logprobs_forward(const Tensor& logits, const Tensor& actions, const Maybe& mask, bool want)
{
    const c10::DeviceGuard guard(logits.device());
    const Tensor z = rows_of(logits);
    const int64_t B = z.size(0), T = z.size(1), V = z.size(2);
    const auto f32 = z.options().dtype(at::kFloat);
    Tensor logp = at::empty({B, T}, f32), entropy = at::empty({B, T}, f32), stats;
    if (want) stats = at::empty({B, T, 3}, f32);
    check(smlvm_token_logprobs_fwd(ptr(z), kind_of(z), z.stride(0), z.stride(1), static_cast<const int64_t*>(ptr(actions)),
                                   static_cast<const uint8_t*>(ptr(mask)), static_cast<float*>(ptr(logp)),
                                   static_cast<float*>(ptr(entropy)), static_cast<float*>(ptr(stats)), B, T, V, stream_of(z)),
          "smlvm_token_logprobs_fwd");
    return {logp, entropy, stats};
}

// (log softmax(logits)[action], entropy) per row without the [.., V] log-probabilities
struct TokenLogprobs : Function<TokenLogprobs> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& actions, const Maybe& mask)
    {
        ctx->set_materialize_grads(false);
        variable_list out = logprobs_forward(logits, actions, mask, true);
        ctx->save_for_backward({logits, actions, out[2], mask ? *mask : Tensor()});
        out.pop_back();
        return out;
    }

    static variable_list backward(AutogradContext* ctx, const variable_list& grads)
    {
        variable_list out(3);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        const variable_list saved = ctx->get_saved_variables();
        const Tensor c = grads[0].defined() ? grads[0].contiguous() : at::zeros_like(grads[1], at::MemoryFormat::Contiguous);
        const Tensor h = grads[1].defined() ? grads[1].contiguous() : Tensor();
        variable_list one = {rows_backward(saved[0], saved[1], saved[3], static_cast<const float*>(ptr(saved[2])),
                                           static_cast<const float*>(ptr(c)), static_cast<const float*>(ptr(h)), Tensor(), Tensor())};
        once(one, {grads[0], grads[1], saved[0]});
        out[0] = one[0];
        return out;
    }
};

std::tuple<Tensor, Tensor> token_logprobs(const Tensor& logits, const Tensor& actions, const Maybe& mask)
{
    no_tangents(logits);
    const bool record = at::GradMode::is_enabled() && wants(logits);
    variable_list out = record ? TokenLogprobs::apply(logits, actions, mask) : logprobs_forward(logits, actions, mask, false);
    return {out[0], out[1]};
}

// The id of the graph capture that the tensor's current stream is part of, 0 outside one.
int64_t capture_of(const Tensor& t)
{
    const c10::DeviceGuard guard(t.device());
    uint64_t id = 0;
    check(smlvm_stream_capture_id(stream_of(t), &id), "smlvm_stream_capture_id");
    return (int64_t)id;
}

// The loss, and in the same pass over the logits its gradient.  The backward hands that buffer on and only launches
// a kernel that returns at once when the incoming gradient is 1 and writes the gradient anew from the
// logits when it is not (scaling the stored one would round 16-bit values twice, and lose what fp16 had already
// flushed to zero).  The buffer is good for one backward pass: a second one (retain_graph), or one recorded into
// another graph capture than the forward (whose replays need not follow a replay of the forward), computes
// into a new tensor.
struct ClippedPolicyLoss : Function<ClippedPolicyLoss> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& actions, const Tensor& old_logp,
                                 const Tensor& advantages, const Maybe& ref_logp, const Maybe& mask, double clip_low, double clip_high,
                                 double kl_coeff, double entropy_coeff, bool mean)
    {
        const c10::DeviceGuard guard(logits.device());
        const bool want = wants(logits);
        const Tensor z = rows_of(logits);
        const int64_t B = z.size(0), T = z.size(1), V = z.size(2), rows = B * T;
        const auto f32 = z.options().dtype(at::kFloat);
        // (every output has memory of its own: one that a caller changes in place must not touch another)
        Tensor logp = at::empty({B, T}, f32), entropy = at::empty({B, T}, f32), kl = at::empty({B, T}, f32), loss = at::empty({}, f32);
        Tensor clipped = at::empty({B, T}, z.options().dtype(at::kBool));
        const Tensor kept = at::empty({rows * 5}, f32);                  // stats [rows, 3], c [rows], h [rows]
        float* const stats = static_cast<float*>(ptr(kept));
        const Tensor dlogits = want ? at::empty({B, T, V}, z.options()) : Tensor();
        const size_t bytes = smlvm_policy_loss_workspace_bytes(rows);
        const Tensor ws = workspace(bytes, z);
        check(smlvm_policy_loss(ptr(z), kind_of(z), z.stride(0), z.stride(1), static_cast<const int64_t*>(ptr(actions)),
                                static_cast<const uint8_t*>(ptr(mask)), static_cast<const float*>(ptr(old_logp)),
                                static_cast<const float*>(ptr(advantages)), static_cast<const float*>(ptr(ref_logp)), (float)clip_low,
                                (float)clip_high, (float)kl_coeff, (float)entropy_coeff, mean ? 1 : 0, static_cast<float*>(ptr(loss)),
                                static_cast<float*>(ptr(logp)), static_cast<float*>(ptr(entropy)), static_cast<float*>(ptr(kl)),
                                static_cast<uint8_t*>(ptr(clipped)), stats, stats + 3 * rows, stats + 4 * rows, ptr(dlogits), B, T, V,
                                ptr(ws), bytes, stream_of(z)),
              "smlvm_policy_loss");
        ctx->set_materialize_grads(false);                               // (no zeros for the statistics' gradients)
        if (want) {
            ctx->save_for_backward({logits, actions, kept, mask ? *mask : Tensor()});
            ctx->saved_data["ready"] = dlogits;
            ctx->saved_data["capture"] = capture_of(z);
        }
        ctx->mark_non_differentiable({logp, entropy, kl, clipped});
        return {loss, logp, entropy, kl, clipped};
    }

    static variable_list backward(AutogradContext* ctx, const variable_list& grads)
    {
        variable_list out(11);
        if (!grads[0].defined()) return out;
        const variable_list saved = ctx->get_saved_variables();
        const Tensor& kept = saved[2];
        const int64_t rows = kept.numel() / 5;
        const float* const stats = static_cast<const float*>(ptr(kept));
        Tensor ready;
        const auto it = ctx->saved_data.find("ready");
        if (it != ctx->saved_data.end()) {
            ready = it->second.toTensor();
            ctx->saved_data.erase(it);
            if (capture_of(kept) != ctx->saved_data["capture"].toInt()) ready = Tensor();
        }
        const Tensor g = grads[0].to(at::kFloat).contiguous();
        variable_list one = {rows_backward(saved[0], saved[1], saved[3], stats, stats + 3 * rows, stats + 4 * rows, g, ready)};
        once(one, {grads[0], saved[0]});
        out[0] = one[0];
        return out;
    }
};

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> clipped_policy_loss(
    const Tensor& logits, const Tensor& actions, const Tensor& old_logp, const Tensor& advantages, const Maybe& ref_logp,
    const Maybe& mask, double clip_low, double clip_high, double kl_coeff, double entropy_coeff, bool mean)
{
    no_tangents(logits, old_logp, advantages, ref_logp);
    const auto out = ClippedPolicyLoss::apply(at::GradMode::is_enabled() ? logits : logits.detach(), actions, old_logp, advantages,
                                              ref_logp, mask, clip_low, clip_high, kl_coeff, entropy_coeff, mean);
    return {out[0], out[1], out[2], out[3], out[4]};
}

// ------------------------------------------------------------------------------------------------ AdamW
constexpr int64_t kBlock = 256;                       // elements that share one scale of an 8-bit state

bool floating(const Tensor& t)
{
    const auto k = t.scalar_type();
    return k == at::kFloat || k == at::kHalf || k == at::kBFloat16;
}

Tensor entry_of(const pybind11::dict& state, const char* key)
{
    PyObject* const o = PyDict_GetItemString(state.ptr(), key);
    return o && THPVariable_Check(o) ? THPVariable_Unpack(o) : Tensor();
}

void adamw_check(const Tensor& p, const Tensor& g)
{
    if (!p.is_cuda() || g.device() != p.device())
        throw NativeError("AdamW: parameters and gradients must be on one GPU (there is no CPU fallback)");
    TORCH_CHECK_TYPE(floating(p) && g.layout() == at::kStrided && floating(g) && g.sizes() == p.sizes(),
                     "AdamW: a gradient must be a dense float32, float16 or bfloat16 tensor of the parameter's shape ", p.sizes(),
                     ", got ", g.scalar_type(), " ", g.sizes(), " (", g.layout(), ")");
}

// One group of parameters: grads[i] None (the parameter is left alone) or its gradient, states[i] its state, numbers[i]
// its number in the rounding hash; tickets: device (its default stream) or (device, stream) -> the kernel's counter word.
// One launch per device, types and kind of state.  True where a launch went into a graph capture.
bool adamw_step(const pybind11::list& params, const pybind11::list& grads, const pybind11::list& states, const pybind11::list& numbers,
                const pybind11::dict& tickets, const pybind11::object& lr, double beta1, double beta2, double eps,
                double weight_decay, int64_t seed)
{
    struct Launch { at::Device device; at::ScalarType p, g; int32_t bits; std::vector<smlvm_adamw_tensor> table; };
    const at::NoGradGuard no_grad;
    const bool rate_tensor = THPVariable_Check(lr.ptr());
    if (rate_tensor) {                                // (the kernel reads it as one float)
        const Tensor& rate = THPVariable_Unpack(lr.ptr());
        TORCH_CHECK_TYPE(rate.scalar_type() == at::kFloat, "AdamW: a tensor lr must be float32, got ", rate.scalar_type());
        TORCH_CHECK_VALUE(rate.numel() == 1, "AdamW: a tensor lr must have one element, got ", rate.sizes());
    }
    std::vector<Launch> launches;
    std::vector<Tensor> keep;                         // alive until the launch: updated parameters and relaid gradients
    const size_t count = params.size();
    keep.reserve(2 * count);
    for (size_t i = 0; i < count; ++i) {
        if (grads[i].is_none()) continue;
        const Tensor p = THPVariable_Unpack(params[i].ptr());
        if (p.numel() == 0) continue;
        Tensor g = pybind11::cast<Tensor>(grads[i]);
        adamw_check(p, g);
        const pybind11::dict state = states[i];
        const Tensor m = entry_of(state, "exp_avg"), step = entry_of(state, "step");
        Tensor v = entry_of(state, "exp_avg_sq"), m_scale, r_scale;
        const bool small = !v.defined();
        if (small) {
            v = entry_of(state, "exp_rms");
            m_scale = entry_of(state, "exp_avg_scale");
            r_scale = entry_of(state, "exp_rms_scale");
        }
        for (const Tensor& t : {m, v, step})
            if (!t.defined() || t.device() != p.device()) throw NativeError("AdamW: a parameter's state is not on its GPU");
        TORCH_CHECK_VALUE(m.sizes() == p.sizes() && v.sizes() == p.sizes() && m.strides() == p.strides() && v.strides() == p.strides(),
                          "AdamW: a parameter changed its shape or memory order after its state was made");
        const auto kind = small ? at::kFloat8_e4m3fn : at::kFloat;
        TORCH_CHECK_TYPE(m.scalar_type() == kind && v.scalar_type() == kind && step.scalar_type() == at::kLong && step.numel() == 1,
                         "AdamW: a parameter's state has other types than this optimiser made it with");
        if (small) {
            const int64_t blocks = (p.numel() + kBlock - 1) / kBlock;
            for (const Tensor& t : {m_scale, r_scale})
                TORCH_CHECK_VALUE(t.defined() && t.device() == p.device() && t.scalar_type() == at::kFloat && t.numel() == blocks &&
                                  t.is_contiguous(), "AdamW: the scales of an 8-bit state do not fit its parameter");
        }
        if (g.strides() != p.strides()) {
            const c10::DeviceGuard guard(p.device());
            g = at::empty_like(p, p.options().dtype(g.scalar_type())).copy_(g);
            keep.push_back(g);
        }
        Launch* to = nullptr;
        for (Launch& l : launches)
            if (l.device == p.device() && l.p == p.scalar_type() && l.g == g.scalar_type() && l.bits == (small ? 8 : 32)) to = &l;
        if (!to) {
            launches.push_back({p.device(), p.scalar_type(), g.scalar_type(), small ? 8 : 32, {}});
            to = &launches.back();
            to->table.reserve(count);
        }
        to->table.push_back({p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), static_cast<float*>(ptr(m_scale)),
                             static_cast<float*>(ptr(r_scale)), static_cast<int64_t*>(step.data_ptr()), p.numel(),
                             pybind11::cast<uint64_t>(numbers[i])});
        keep.push_back(p);
    }
    bool captured = false;
    for (const Launch& l : launches) {
        const c10::DeviceGuard guard(l.device);
        const c10::hip::HIPStream stream = c10::hip::getCurrentHIPStream(l.device.index());
        uint64_t capture = 0;
        check(smlvm_stream_capture_id(stream.stream(), &capture), "smlvm_stream_capture_id");
        Tensor rate;
        double number = 0.0;
        if (rate_tensor) {
            rate = THPVariable_Unpack(lr.ptr());
            if (rate.device() != l.device) {
                TORCH_CHECK_VALUE(!rate.is_cuda(), "AdamW: a tensor lr must be on the parameters' device");
                TORCH_CHECK(!capture, "AdamW: a captured step reads a tensor lr at every replay: it must be on the parameters' device");
                number = rate.item<double>();
                rate = Tensor();
            }
        } else {
            number = pybind11::cast<double>(lr);
        }
        captured |= capture != 0;
        Tensor ticket;                                // (a word per stream: steps on two of them may overlap)
        if (!capture) {
            pybind11::object key = pybind11::cast(l.device);
            if (stream.id() != 0) key = pybind11::make_tuple(key, stream.id());
            if (!tickets.contains(key)) tickets[key] = at::zeros({1}, at::TensorOptions(l.device).dtype(at::kInt));
            ticket = pybind11::cast<Tensor>(tickets[key]);
        }
        check(smlvm_adamw_step(l.table.data(), (int32_t)l.table.size(), kind_of(l.p), kind_of(l.g), l.bits, beta1, beta2, (float)eps, (float)number, static_cast<const float*>(ptr(rate)), (float)weight_decay,
                               (uint32_t)seed, static_cast<uint32_t*>(ptr(ticket)), stream.stream()),
              "smlvm_adamw_step");
    }
    // (a graph that had saved a parameter's old value finds out)
    for (const Tensor& p : keep) if (!p.is_inference()) torch::autograd::impl::bump_version(p);
    return captured;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    pybind11::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const NativeError& e) {
            PyErr_SetString(pybind11::module_::import("lvmhelpers._native").attr("NativeError").ptr(), e.what());
        }
    });
    m.def("linear_act", &linear_act);
    m.def("token_logprobs", &token_logprobs);
    m.def("clipped_policy_loss", &clipped_policy_loss);
    m.def("adamw_step", &adamw_step);
}
