// The context operators (attention, gated feed-forward, residual norm) as dispatcher ops with their autograd nodes in C++: a small call is
// bounded by what happens on the host around its launches, and a backward that never enters Python costs the engine no hand-over of the
// interpreter.  Same C-ABI functions underneath as every other op; arguments are checked by the Python functions that call these
// (attention.py, feedforward.py, norms.py), here only what memory safety needs.  Host-only C++.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/autograd.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <unordered_set>
#include <vector>

#include "../../include/equigspr.h"

namespace {

using OptTensor = std::optional<at::Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

hipStream_t stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
const void* cptr(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
at::Tensor value(const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); }

void check(int rc, const char* what) { TORCH_CHECK(rc == 0, "equigspr::", what, ": ", equigspr_last_error(), " (code ", rc, ")"); }
int dtype_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return EQUIGSPR_F32;
        case at::kBFloat16: return EQUIGSPR_BF16;
        case at::kHalf: return EQUIGSPR_F16;
        default: TORCH_CHECK(false, "equigspr: expected float32, bfloat16 or float16, got ", t.scalar_type());
    }
}
// sizes that the C entries count in 32 bits
bool counted(int64_t n) { return n < (1ll << 31); }
// on the GPU, of one type and device with `like`, and (dense) contiguous
void need(const at::Tensor& t, const at::Tensor& like, const char* name, bool dense) {
    if (!t.defined()) return;
    TORCH_CHECK(t.is_cuda(), "equigspr: ", name, " must live on the GPU (there is no CPU path)");
    TORCH_CHECK(t.scalar_type() == like.scalar_type() && t.device() == like.device(), "equigspr: ", name, " differs in dtype or device");
    TORCH_CHECK(!dense || t.is_contiguous(), "equigspr: ", name, " must be contiguous");
}

// Whether a backward that is recorded into a hipGraph from here on would reach into work of another stream: `t` -- or anything before it in
// its autograd graph, down to the leaves' gradient accumulators, which an eager graph of the same leaves keeps alive -- was built on a stream
// that is not being captured.  The autograd engine would synchronise with that stream during the capture, which ends the process; the ops
// raise instead.  Walked only while a call is being recorded.
bool node_on_other_stream(torch::autograd::Node& node, hipStream_t now) {
    const auto stream = node.stream();
    if (!stream.has_value()) return false;
    const c10::hip::HIPStreamMasqueradingAsCUDA other(*stream);      // autograd's streams carry the masqueraded device type
    if (other.stream() == now) return false;
    if (other.stream() == nullptr) return true;                     // the default stream is never part of a capture
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(other.stream(), &status) != hipSuccess) { (void)hipGetLastError(); return true; }
    return status != hipStreamCaptureStatusActive;
}
bool grad_lives_on_other_stream(const at::Tensor& t) {
    if (!t.defined() || !t.is_cuda() || !t.requires_grad()) return false;
    const hipStream_t now = stream_of(t);
    const std::shared_ptr<torch::autograd::Node> first = t.grad_fn() ? t.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(t);
    std::vector<torch::autograd::Node*> open = {first.get()};        // first keeps everything behind it alive
    std::unordered_set<torch::autograd::Node*> seen;
    while (!open.empty()) {
        torch::autograd::Node* const node = open.back();
        open.pop_back();
        if (!node || !seen.insert(node).second) continue;
        if (node_on_other_stream(*node, now)) return true;
        for (const auto& edge : node->next_edges()) open.push_back(edge.function.get());
    }
    return false;
}
// true if one of the inputs wants a gradient; refuses a capture that would end the process, and tangents, which the output would lose
bool training(std::initializer_list<at::Tensor> inputs) {
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode())
        for (const auto& t : inputs)
            TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), "equigspr: the context operators have no forward-mode derivative");
    if (!at::GradMode::is_enabled()) return false;
    bool any = false;
    at::Tensor one;
    for (const auto& t : inputs)
        if (t.defined() && t.requires_grad()) { any = true; one = t; }
    if (!any) return false;
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    const hipStream_t now = stream_of(one);
    if (now != nullptr && hipStreamIsCapturing(now, &status) == hipSuccess && status == hipStreamCaptureStatusActive) {
        int i = 0;
        for (const auto& t : inputs) {
            TORCH_CHECK(!grad_lives_on_other_stream(t), "input ", i, " hangs on an autograd graph that was built on another stream and is still alive: drop that "
                        "graph's outputs (or run it on the capturing stream) before recording this call into a hipGraph");
            ++i;
        }
    }
    return true;
}
// gradients are differentiable once: under create_graph they carry a node that raises when it is reached
variable_list once(variable_list grads, const char* what) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list some;
    for (auto& g : grads)
        if (g.defined()) { g.set_requires_grad(true); some.push_back(g); }
    if (some.empty()) return grads;
    const auto node = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " is differentiable once", (int64_t)some.size());
    some = (*node)(std::move(some));
    size_t k = 0;
    for (auto& g : grads)
        if (g.defined()) g = some[k++];
    return grads;
}

// ------------------------------------------------------------------------------------------------ attention
int64_t stride_of(const at::Tensor& t, int axis) { return t.size(axis) > 1 ? t.stride(axis) : 0; }
equigspr_attention_tensor rows_of(const at::Tensor& t) { return {const_cast<void*>(t.const_data_ptr()), stride_of(t, 0), stride_of(t, 1), stride_of(t, 2)}; }

equigspr_attention describe(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& q_lens, const at::Tensor& kv_lens, const at::Tensor& mask,
                            bool causal, double scale) {
    equigspr_attention d = {};
    d.dtype = dtype_code(q);
    for (int i = 0; i < 4; ++i) TORCH_CHECK(counted(q.size(i)) && counted(k.size(i)), "equigspr::cloud_attention: sizes out of range");
    d.batch = (int32_t)q.size(0); d.nq = (int32_t)q.size(1); d.nk = (int32_t)k.size(1);
    d.heads = (int32_t)q.size(2); d.kv_heads = (int32_t)k.size(2); d.dim = (int32_t)q.size(3);
    d.causal = causal;
    d.scale = (float)scale;
    d.q = rows_of(q); d.k = rows_of(k); d.v = rows_of(v);
    d.q_lens = (const int32_t*)cptr(q_lens); d.kv_lens = (const int32_t*)cptr(kv_lens);
    d.key_mask = (const uint8_t*)cptr(mask);
    d.mask_stride = mask.defined() ? mask.stride(0) : 0;
    return d;
}
at::Tensor floats(int64_t n, const at::Tensor& like) { return at::empty({n}, like.options().dtype(at::kFloat)); }

// out, and, training, out_low (16-bit types) and lse
std::tuple<at::Tensor, at::Tensor, at::Tensor> attention_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& q_lens,
                                                                 const at::Tensor& kv_lens, const at::Tensor& mask, bool causal, double scale, bool train) {
    const c10::DeviceGuard guard(q.device());
    const auto d = describe(q, k, v, q_lens, kv_lens, mask, causal, scale);
    const int64_t n = equigspr_attention_work_size(&d);
    TORCH_CHECK(n >= 0, "equigspr::attention_forward: ", equigspr_last_error());
    const at::Tensor work = n > 0 ? floats(n, q) : at::Tensor(), out = at::empty(q.sizes(), q.options());
    const at::Tensor low = train && q.scalar_type() != at::kFloat ? at::empty(q.sizes(), q.options()) : at::Tensor();
    const at::Tensor lse = train ? floats(q.size(0) * q.size(1) * q.size(2), q) : at::Tensor();
    check(equigspr_attention_forward(&d, ptr(out), ptr(low), (float*)ptr(lse), (float*)ptr(work), stream_of(q)), "attention_forward");
    return {out, low, lse};
}

struct AttentionFn : torch::autograd::Function<AttentionFn> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptTensor& q_lens, const OptTensor& kv_lens,
                              const OptTensor& mask, bool causal, double scale) {
        auto [out, low, lse] = attention_forward(q, k, v, value(q_lens), value(kv_lens), value(mask), causal, scale, true);
        ctx->save_for_backward({q, k, v, value(q_lens), value(kv_lens), value(mask), out, low, lse});
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["scale"] = scale;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        const at::Tensor &q = s[0], &k = s[1], &v = s[2];
        const c10::DeviceGuard guard(q.device());
        const auto d = describe(q, k, v, s[3], s[4], s[5], ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble());
        at::Tensor go = g[0];
        const bool near = (stride_of(go, 1) + stride_of(go, 2)) * 128 * (int64_t)go.element_size() < (1ll << 31);
        if (!near || (go.size(3) > 1 && go.stride(3) != 1)) go = go.contiguous();
        const auto grad = [&](int i, const at::Tensor& t) { return ctx->needs_input_grad(i) ? at::empty(t.sizes(), t.options()) : at::Tensor(); };
        const at::Tensor gq = grad(0, q), gk = grad(1, k), gv = grad(2, v), work = floats(equigspr_attention_backward_work_size(&d), q);
        const auto gr = rows_of(go);
        check(equigspr_attention_backward(&d, cptr(s[6]), cptr(s[7]), (const float*)cptr(s[8]), &gr, (float*)ptr(work), ptr(gq), ptr(gk), ptr(gv), stream_of(q)),
              "attention_backward");
        auto out = once({gq, gk, gv}, "cloud_attention");
        out.resize(8);
        return out;
    }
};

at::Tensor cloud_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptTensor& q_lens, const OptTensor& kv_lens, const OptTensor& mask,
                           bool causal, double scale) {
    need(q, q, "q", false);
    need(k, q, "k", false);
    need(v, q, "v", false);
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.sizes() == k.sizes() && k.size(0) == q.size(0) && k.size(3) == q.size(3), "equigspr::cloud_attention: shapes do not belong together");
    for (const auto* t : {&q, &k, &v}) TORCH_CHECK(t->size(3) <= 1 || t->stride(3) == 1, "equigspr::cloud_attention: the last dimension must be dense");
    for (const auto* t : {&q_lens, &kv_lens})
        TORCH_CHECK(!t->has_value() || ((*t)->is_cuda() && (*t)->device() == q.device() && (*t)->scalar_type() == at::kInt && (*t)->is_contiguous() && (*t)->numel() == q.size(0)),
                    "equigspr::cloud_attention: lengths must be int32 [B] on the inputs' device");
    TORCH_CHECK(!mask.has_value() || (mask->is_cuda() && mask->device() == q.device() && mask->scalar_type() == at::kBool && mask->dim() == 2 && mask->size(0) == q.size(0) &&
                                      mask->size(1) == k.size(1) && (mask->size(1) <= 1 || mask->stride(1) == 1)),
                "equigspr::cloud_attention: key_mask must be bool [B, Nk] with dense rows");
    if (training({q, k, v})) return AttentionFn::apply(q, k, v, q_lens, kv_lens, mask, causal, scale);
    return std::get<0>(attention_forward(q, k, v, value(q_lens), value(kv_lens), value(mask), causal, scale, false));
}

// ------------------------------------------------------------------------------------------------ gated feed-forward
equigspr_gated_feed_forward describe(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, const at::Tensor& bg, const at::Tensor& bu,
                                     const at::Tensor& bd, int64_t act) {
    equigspr_gated_feed_forward d = {};
    d.dtype = dtype_code(x);
    d.activation = (int32_t)act;
    TORCH_CHECK(counted(x.size(0)) && counted(x.size(1)) && counted(wg.size(0)) && counted(wd.size(0)), "equigspr::gated_feed_forward: sizes out of range");
    d.rows = (int32_t)x.size(0); d.width = (int32_t)x.size(1); d.hidden = (int32_t)wg.size(0); d.out = (int32_t)wd.size(0);
    d.x = cptr(x); d.w_gate = cptr(wg); d.w_up = cptr(wu); d.w_down = cptr(wd);
    d.b_gate = cptr(bg); d.b_up = cptr(bu); d.b_down = cptr(bd);
    return d;
}

// y, h and, training, both projections
std::tuple<at::Tensor, at::Tensor, at::Tensor> feed_forward_forward(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, const at::Tensor& bg,
                                                                    const at::Tensor& bu, const at::Tensor& bd, int64_t act, bool train) {
    const c10::DeviceGuard guard(x.device());
    const auto d = describe(x, wg, wu, wd, bg, bu, bd, act);
    const int64_t n = equigspr_gated_feed_forward_work_size(&d);
    TORCH_CHECK(n >= 0, "equigspr::gated_feed_forward_forward: ", equigspr_last_error());
    const at::Tensor work = n > 0 ? floats(n, x) : at::Tensor(), y = at::empty({x.size(0), wd.size(0)}, x.options()), h = at::empty({x.size(0), wg.size(0)}, x.options());
    const at::Tensor zu = train ? at::empty({x.size(0), 2 * wg.size(0)}, x.options().dtype(at::kFloat)) : at::Tensor();
    check(equigspr_gated_feed_forward_forward(&d, ptr(y), ptr(h), (float*)ptr(zu), (float*)ptr(work), stream_of(x)), "gated_feed_forward_forward");
    return {y, h, zu};
}

struct FeedForwardFn : torch::autograd::Function<FeedForwardFn> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, const OptTensor& bg, const OptTensor& bu,
                              const OptTensor& bd, int64_t act) {
        auto [y, h, zu] = feed_forward_forward(x, wg, wu, wd, value(bg), value(bu), value(bd), act, true);
        ctx->save_for_backward({x, wg, wu, wd, h, zu});
        ctx->saved_data["act"] = act;
        ctx->saved_data["biases"] = (int64_t)(value(bg).defined() | value(bu).defined() << 1 | value(bd).defined() << 2);
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        const at::Tensor &x = s[0], &wg = s[1], &wd = s[3];
        const c10::DeviceGuard guard(x.device());
        const auto d = describe(x, wg, s[2], wd, at::Tensor(), at::Tensor(), at::Tensor(), ctx->saved_data["act"].toInt());
        const int64_t rows = x.size(0), hidden = wg.size(0), out = wd.size(0);
        const at::Tensor gy = g[0].contiguous();
        // autograd counts an edge for every tensor that was given
        const int64_t biases = ctx->saved_data["biases"].toInt();
        bool wanted[7];
        for (int i = 0, edge = 0; i < 7; ++i) wanted[i] = (i < 4 || (biases >> (i - 4) & 1)) && ctx->needs_input_grad(edge++);
        const auto want = [&](int i) { return wanted[i]; };
        const auto grad = [&](bool on, at::IntArrayRef shape) { return !on ? at::Tensor() : rows ? at::empty(shape, x.options()) : at::zeros(shape, x.options()); };
        const at::Tensor gx = grad(want(0), x.sizes()), gw = grad(want(1) || want(2), {2 * hidden, x.size(1)}), gd = grad(want(3), wd.sizes());
        const at::Tensor gb = grad(want(4) || want(5), {2 * hidden}), gbd = grad(want(6), {out}), dzu = at::empty({rows, 2 * hidden}, x.options());
        const at::Tensor work = floats(std::max<int64_t>(1, equigspr_gated_feed_forward_backward_work_size(&d)), x);
        const equigspr_gated_feed_forward_grads o = {ptr(gx), ptr(gw), ptr(gd), ptr(gb), ptr(gbd)};
        check(equigspr_gated_feed_forward_backward(&d, cptr(gy), (const float*)cptr(s[5]), cptr(s[4]), ptr(dzu), (float*)ptr(work), &o, stream_of(x)), "gated_feed_forward_backward");
        const auto half = [&](const at::Tensor& t, int i, int64_t at) { return want(i) ? t.narrow(0, at, hidden) : at::Tensor(); };
        auto r = once({gx, half(gw, 1, 0), half(gw, 2, hidden), gd, half(gb, 4, 0), half(gb, 5, hidden), gbd}, "gated_feed_forward");
        r.resize(8);
        return r;
    }
};

at::Tensor gated_feed_forward(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, const OptTensor& bg, const OptTensor& bu, const OptTensor& bd,
                              int64_t act) {
    need(x, x, "x", true);
    for (const auto* t : {&wg, &wu, &wd}) need(*t, x, "a weight", true);
    for (const auto* t : {&bg, &bu, &bd}) need(value(*t), x, "a bias", true);
    TORCH_CHECK(x.dim() == 2 && wg.dim() == 2 && wd.dim() == 2 && wu.sizes() == wg.sizes() && wg.size(1) == x.size(1) && wd.size(1) == wg.size(0), "equigspr::gated_feed_forward: shapes do not belong together");
    TORCH_CHECK((!bg.has_value() || bg->numel() == wg.size(0)) && (!bu.has_value() || bu->numel() == wg.size(0)) && (!bd.has_value() || bd->numel() == wd.size(0)),
                "equigspr::gated_feed_forward: a bias has the wrong size");
    if (training({x, wg, wu, wd, value(bg), value(bu), value(bd)})) return FeedForwardFn::apply(x, wg, wu, wd, bg, bu, bd, act);
    return std::get<0>(feed_forward_forward(x, wg, wu, wd, value(bg), value(bu), value(bd), act, false));
}

// ------------------------------------------------------------------------------------------------ residual norm
struct NormRest { bool rms; double eps, factor; int64_t gate_rows; };
equigspr_residual_norm describe(const variable_list& t, const NormRest& r) {      // x, f, pre_weight, pre_bias, post_weight, post_bias, gate, scale
    equigspr_residual_norm d = {};
    const at::Tensor& x = t[0];
    d.dtype = dtype_code(x);
    TORCH_CHECK(counted(x.size(-1)), "equigspr::residual_norm: width out of range");
    d.width = (int32_t)x.size(-1);
    d.rms = r.rms;
    d.rows = x.numel() / x.size(-1);
    d.gate_rows = r.gate_rows;
    d.eps = (float)r.eps; d.factor = (float)r.factor;
    d.x = cptr(x); d.f = cptr(t[1]); d.gate = cptr(t[6]);
    d.pre_weight = (const float*)cptr(t[2]); d.pre_bias = (const float*)cptr(t[3]);
    d.post_weight = (const float*)cptr(t[4]); d.post_bias = (const float*)cptr(t[5]);
    d.scale = (const float*)cptr(t[7]);
    return d;
}
// y (undefined without f) and u (undefined without the second norm)
variable_list norm_forward(const variable_list& t, const NormRest& r) {
    const at::Tensor& x = t[0];
    const c10::DeviceGuard guard(x.device());
    const auto d = describe(t, r);
    const at::Tensor y = t[1].defined() ? at::empty(x.sizes(), x.options()) : at::Tensor(), u = t[2].defined() ? at::empty(x.sizes(), x.options()) : at::Tensor();
    check(equigspr_residual_norm_forward(&d, ptr(y), ptr(u), stream_of(x)), "residual_norm_forward");
    return {y, u};
}

struct ResidualNormFn : torch::autograd::Function<ResidualNormFn> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& f, const OptTensor& pre_w, const OptTensor& pre_b, const OptTensor& post_w,
                                 const OptTensor& post_b, const OptTensor& gate, const OptTensor& scale, bool rms, double eps, double factor, int64_t gate_rows) {
        const variable_list t = {x, value(f), value(pre_w), value(pre_b), value(post_w), value(post_b), value(gate), value(scale)};
        ctx->set_materialize_grads(false);
        ctx->save_for_backward(t);
        ctx->saved_data["rms"] = rms;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["factor"] = factor;
        ctx->saved_data["gate_rows"] = gate_rows;
        auto out = norm_forward(t, {rms, eps, factor, gate_rows});
        variable_list some;
        for (auto& o : out)
            if (o.defined()) some.push_back(o);
        ctx->saved_data["has_y"] = out[0].defined();
        return some;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto t = ctx->get_saved_variables();
        const at::Tensor& x = t[0];
        const c10::DeviceGuard guard(x.device());
        const auto d = describe(t, {ctx->saved_data["rms"].toBool(), ctx->saved_data["eps"].toDouble(), ctx->saved_data["factor"].toDouble(), ctx->saved_data["gate_rows"].toInt()});
        const bool has_y = ctx->saved_data["has_y"].toBool();
        const auto dense = [](const at::Tensor& v) { return v.defined() ? v.contiguous() : v; };
        const at::Tensor gy = has_y ? dense(g[0]) : at::Tensor(), gu = t[2].defined() ? dense(g[has_y ? 1 : 0]) : at::Tensor();
        variable_list got(8);
        for (int i = 0, edge = 0; i < 8; ++i)                       // autograd counts an edge for every tensor that was given
            if (t[i].defined() && ctx->needs_input_grad(edge++)) got[i] = x.numel() ? at::empty(t[i].sizes(), t[i].options()) : at::zeros(t[i].sizes(), t[i].options());
        const at::Tensor work = floats(std::max<int64_t>(1, equigspr_residual_norm_backward_work_size(&d)), x);
        const equigspr_residual_norm_grads o = {ptr(got[0]), ptr(got[1]), ptr(got[6]), (float*)ptr(got[4]), (float*)ptr(got[5]), (float*)ptr(got[2]), (float*)ptr(got[3]), (float*)ptr(got[7])};
        check(equigspr_residual_norm_backward(&d, cptr(gy), cptr(gu), (float*)ptr(work), &o, stream_of(x)), "residual_norm_backward");
        got = once(std::move(got), "residual_norm");
        got.resize(12);
        return got;
    }
};

std::tuple<at::Tensor, at::Tensor> residual_norm(const at::Tensor& x, const OptTensor& f, const OptTensor& pre_w, const OptTensor& pre_b, const OptTensor& post_w, const OptTensor& post_b,
                                                 const OptTensor& gate, const OptTensor& scale, bool rms, double eps, double factor, int64_t gate_rows) {
    need(x, x, "x", true);
    need(value(f), x, "f", true);
    need(value(gate), x, "gate", true);
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && (!f.has_value() || f->sizes() == x.sizes()), "equigspr::residual_norm: f must be shaped like x");
    const int64_t width = x.size(-1), rows = x.numel() / width;
    for (const auto* t : {&pre_w, &pre_b, &post_w, &post_b, &scale})
        TORCH_CHECK(!t->has_value() || ((*t)->is_cuda() && (*t)->device() == x.device() && (*t)->scalar_type() == at::kFloat && (*t)->is_contiguous() && (*t)->numel() == width),
                    "equigspr::residual_norm: weights, biases and scale must be float32 [width] on the inputs' device");
    TORCH_CHECK(gate_rows >= 1 && (!gate.has_value() || rows == 0 || (rows % gate_rows == 0 && gate->numel() == rows / gate_rows * width)), "equigspr::residual_norm: the gate does not fit x");
    variable_list out;
    if (training({x, value(f), value(pre_w), value(pre_b), value(post_w), value(post_b), value(gate), value(scale)})) {
        auto some = ResidualNormFn::apply(x, f, pre_w, pre_b, post_w, post_b, gate, scale, rms, eps, factor, gate_rows);
        size_t k = 0;
        out = {f.has_value() ? some[k++] : at::Tensor(), pre_w.has_value() ? some[k] : at::Tensor()};
    } else {
        out = norm_forward({x, value(f), value(pre_w), value(pre_b), value(post_w), value(post_b), value(gate), value(scale)}, {rms, eps, factor, gate_rows});
    }
    return {out[0], out[1]};
}
}  // namespace

TORCH_LIBRARY_FRAGMENT(equigspr, m) {
    m.def("cloud_attention(Tensor q, Tensor k, Tensor v, Tensor? q_lens, Tensor? kv_lens, Tensor? key_mask, bool causal, float scale) -> Tensor", &cloud_attention);
    m.def("gated_feed_forward(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, Tensor? b_gate, Tensor? b_up, Tensor? b_down, int activation) -> Tensor", &gated_feed_forward);
    m.def("residual_norm(Tensor x, Tensor? f, Tensor? pre_weight, Tensor? pre_bias, Tensor? post_weight, Tensor? post_bias, Tensor? gate, Tensor? scale, bool rms, float eps, "
          "float factor, int gate_rows) -> (Tensor, Tensor)", &residual_norm);
}
