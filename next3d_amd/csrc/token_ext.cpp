// Host side of the token operators (layer_norm, rotary, attention) in C++: buffers, descriptors and autograd nodes around the C entry points of libn3d.so.
// A Python autograd node costs some 45 us a step more than one in C++ (the engine runs it on another thread, which has to take the interpreter's lock) —
// more than most of these launches.  Arguments arrive checked (torch_utils/ops/*.py); `bind` hands over the entry points of the library that _lib.py has
// loaded, so there is one library and one place that loads it.
#include <ATen/ATen.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/n3d.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<Tensor> Opt;

struct Library {
    decltype(&n3d_last_error) last_error = nullptr;
    decltype(&n3d_layer_norm) layer_norm = nullptr;
    decltype(&n3d_layer_norm_bwd_workspace) layer_norm_bwd_workspace = nullptr;
    decltype(&n3d_layer_norm_bwd) layer_norm_bwd = nullptr;
    decltype(&n3d_rotary) rotary = nullptr;
    decltype(&n3d_attention_workspace) attention_workspace = nullptr;
    decltype(&n3d_attention) attention = nullptr;
    decltype(&n3d_attention_bwd_workspace) attention_bwd_workspace = nullptr;
    decltype(&n3d_attention_bwd) attention_bwd = nullptr;
} lib;

template <typename F>
void set(F& f, size_t address) { f = reinterpret_cast<F>(address); }

void bind(const std::vector<size_t>& a) {
    if (a.size() != 9) throw std::runtime_error("token_ext: nine entry points expected");
    set(lib.last_error, a[0]);
    set(lib.layer_norm, a[1]);
    set(lib.layer_norm_bwd_workspace, a[2]);
    set(lib.layer_norm_bwd, a[3]);
    set(lib.rotary, a[4]);
    set(lib.attention_workspace, a[5]);
    set(lib.attention, a[6]);
    set(lib.attention_bwd_workspace, a[7]);
    set(lib.attention_bwd, a[8]);
}

void check(int64_t rc) {
    if (rc < 0) throw std::runtime_error(std::string("libn3d: ") + lib.last_error());
}

// The device of a call's tensors, whatever the current one is, and torch's current stream there.  Nothing here is recorded by autograd.
struct Scope {
    c10::DeviceGuard device;
    at::AutoDispatchBelowADInplaceOrView below;
    n3d_stream_t stream;
    explicit Scope(const Tensor& t) : device(t.device()), stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream()) {}
};

int code(const Tensor& t) { return t.scalar_type() == at::kHalf ? N3D_F16 : t.scalar_type() == at::kBFloat16 ? N3D_BF16 : N3D_F32; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor get(const Opt& t) { return t ? *t : Tensor(); }
Tensor dense(const Tensor& like) { return at::empty(like.sizes(), like.options().memory_format(c10::MemoryFormat::Contiguous)); }
// What a call of the library cannot serve, and would answer wrongly without a word: a tracer would record the empty output and not the kernel that fills it,
// a tangent would be dropped, a tensor that holds no memory would pass for an absent one.
void refuse(const char* op, std::initializer_list<const Tensor*> ts) {
    const std::string name = op;
    if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY))
        throw std::runtime_error(name + ": cannot be traced");
    const bool tangents = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    for (const Tensor* t : ts) {
        if (!t->defined()) continue;
        if (tangents && t->_fw_grad(0).defined()) throw std::runtime_error(name + ": no forward-mode derivative");
        if (t->numel() && !t->const_data_ptr()) throw std::runtime_error(name + ": a tensor without memory of its own");
    }
}
bool wants_grad(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// Gradients of a backward pass that records itself (create_graph): they refuse to be differentiated again instead of being constants without saying so.
variable_list once(variable_list grads, const char* op) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list given, out;
    for (const Tensor& g : grads)
        if (g.defined()) given.push_back(g.detach().requires_grad_());
    if (given.empty()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(op) + ": differentiable once only", (int64_t)given.size());
    given = (*error)(std::move(given));
    size_t at = 0;
    for (const Tensor& g : grads) out.push_back(g.defined() ? given[at++] : Tensor());
    return out;
}

// ------------------------------------------------------------------------------------------------------------------------------ layer norm
// [rows, C] with dense channels: a view where the strides allow it
Tensor rows_of(const Tensor& x) {
    const int64_t c = x.size(-1);
    const Tensor r = x.dim() == 2 ? x : x.reshape({x.numel() / c, c});
    return c == 1 || r.stride(1) == 1 ? r : r.contiguous();
}

std::pair<Tensor, Tensor> layer_norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, bool want_stats) {
    Scope scope(x);
    const Tensor x2 = rows_of(x), y = dense(x);
    const int64_t rows = x2.size(0), c = x2.size(1);
    Tensor stats;
    float* s = nullptr;
    if (want_stats) {
        stats = at::empty({2, rows}, x.options().dtype(at::kFloat));              // mean, rstd
        s = stats.data_ptr<float>();
    }
    check(lib.layer_norm(x2.data_ptr(), ptr(w), ptr(b), y.data_ptr(), s, s ? s + rows : nullptr, rows, (int)c, x2.stride(0), code(x),
                         w.defined() ? code(w) : b.defined() ? code(b) : N3D_F32, (float)eps, scope.stream));
    return {y, stats};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Opt& weight, const Opt& bias, double eps) {
        const Tensor w = get(weight), b = get(bias);
        const auto [y, stats] = layer_norm_forward(x, w, b, eps, true);
        ctx->save_for_backward({x, w, b, stats});
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &stats = saved[3];
        Tensor dx, dw, db;
        {
            Scope scope(x);
            const Tensor x2 = rows_of(x), dy = rows_of(grads[0].resolve_neg());
            const int64_t rows = x2.size(0), c = x2.size(1);
            if (ctx->needs_input_grad(0)) dx = dense(x);
            // (absent tensors have no edge: the bias comes right behind the weight, or behind x)
            if (w.defined() && ctx->needs_input_grad(1)) dw = at::empty({c}, w.options());
            if (b.defined() && ctx->needs_input_grad(w.defined() ? 2 : 1)) db = at::empty({c}, b.options());
            if (rows) {
                Tensor ws;
                if (dw.defined() || db.defined()) ws = at::empty({lib.layer_norm_bwd_workspace(rows, (int)c, code(x))}, stats.options());
                const float* s = stats.data_ptr<float>();
                check(lib.layer_norm_bwd(dy.data_ptr(), x2.data_ptr(), ptr(w), s, s + rows, ptr(dx), ptr(dw), ptr(db), (float*)ptr(ws), rows, (int)c, x2.stride(0),
                                         dy.stride(0), code(x), w.defined() ? code(w) : b.defined() ? code(b) : N3D_F32, scope.stream));
            } else {
                if (dw.defined()) dw.zero_();
                if (db.defined()) db.zero_();
            }
        }
        return once({dx, dw, db, Tensor()}, "layer_norm");
    }
};

Tensor layer_norm(const Tensor& x, const Opt& weight, const Opt& bias, double eps) {
    Tensor w = get(weight), b = get(bias);
    refuse("layer_norm", {&x, &w, &b});
    if (w.defined()) w = w.contiguous();
    if (b.defined()) b = b.contiguous();
    if (wants_grad({&x, &w, &b})) return LayerNorm::apply(x, w.defined() ? Opt(w) : Opt(), b.defined() ? Opt(b) : Opt(), eps);
    return layer_norm_forward(x, w, b, eps, false).first;
}

// ---------------------------------------------------------------------------------------------------------------------------------- rotary
struct RotaryPlan {
    std::vector<int64_t> sections;
    double base;
    bool interleaved, shared;
};

std::pair<Tensor, Tensor> turn(Tensor q, Tensor k, const Tensor& positions, const RotaryPlan& plan, bool inverse) {
    const Tensor first = q.defined() ? q : k;
    Scope scope(first);
    Tensor yq, yk;
    n3d_rotary_desc d = {};
    if (q.defined()) {
        if (q.stride(3) != 1) q = q.contiguous();
        yq = dense(q);
        d.q = q.data_ptr();
        d.out_q = yq.data_ptr();
        d.heads_q = (int)q.size(2);
        for (int i = 0; i < 3; ++i) d.q_strides[i] = q.stride(i);
    }
    if (k.defined()) {
        if (k.stride(3) != 1) k = k.contiguous();
        yk = dense(k);
        d.k = k.data_ptr();
        d.out_k = yk.data_ptr();
        d.heads_k = (int)k.size(2);
        for (int i = 0; i < 3; ++i) d.k_strides[i] = k.stride(i);
    }
    d.positions = positions.data_ptr();
    d.pos_batch_stride = positions.dim() == 3 && positions.size(0) > 1 ? positions.stride(0) : 0;
    d.pos_token_stride = positions.stride(-2);
    d.base = plan.base;
    d.B = (int)first.size(0);
    d.L = (int)first.size(1);
    d.D = (int)first.size(3);
    d.axes = (int)plan.sections.size();
    for (int a = 0; a < d.axes && a < 4; ++a) d.sections[a] = (int)plan.sections[a];
    d.dtype = code(first);
    d.pos_type = positions.scalar_type() == at::kFloat ? 0 : positions.scalar_type() == at::kInt ? 1 : 2;
    d.interleaved = plan.interleaved;
    d.shared_ladder = plan.shared;
    d.inverse = inverse;
    check(lib.rotary(&d, scope.stream));
    return {yq, yk};
}

struct Rotary : torch::autograd::Function<Rotary> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Opt& k, const Tensor& positions, const RotaryPlan& plan) {
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({positions});
        ctx->saved_data["sections"] = plan.sections;
        ctx->saved_data["base"] = plan.base;
        ctx->saved_data["form"] = (int64_t)(plan.interleaved + 2 * plan.shared);
        const auto [yq, yk] = turn(q, get(k), positions, plan, false);
        return yk.defined() ? variable_list{yq, yk} : variable_list{yq};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const int64_t form = ctx->saved_data["form"].toInt();
        const RotaryPlan plan = {ctx->saved_data["sections"].toIntVector(), ctx->saved_data["base"].toDouble(), (form & 1) != 0, (form & 2) != 0};
        const Tensor positions = ctx->get_saved_variables()[0];
        Tensor dq = grads[0], dk = grads.size() > 1 ? grads[1] : Tensor();
        if (dq.defined() && !ctx->needs_input_grad(0)) dq = Tensor();
        if (dk.defined() && !ctx->needs_input_grad(1)) dk = Tensor();
        if (dq.defined()) dq = dq.resolve_neg();
        if (dk.defined()) dk = dk.resolve_neg();
        if (dq.defined() || dk.defined()) std::tie(dq, dk) = turn(dq, dk, positions, plan, true);
        return once({dq, dk, Tensor(), Tensor()}, "rotary");
    }
};

std::tuple<Tensor, Opt> rotary(const Tensor& q, const Opt& k, const Tensor& positions, const std::vector<int64_t>& sections, double base, bool interleaved, bool shared) {
    const Tensor k_ = get(k);
    refuse("rotary", {&q, &k_, &positions});
    const Tensor pos = positions.stride(-1) == 1 ? positions : positions.contiguous();
    const RotaryPlan plan = {sections, base, interleaved, shared};
    if (wants_grad({&q, &k_})) {
        variable_list y = Rotary::apply(q, k, pos, plan);
        return {y[0], y.size() > 1 ? Opt(y[1]) : Opt()};
    }
    auto [yq, yk] = turn(q, k_, pos, plan, false);
    return {yq, yk.defined() ? Opt(yk) : Opt()};
}

// ------------------------------------------------------------------------------------------------------------------------------- attention
// t [B, L, H, D] itself if the kernels can read it where it lies — dense channels, strides of whole 16-byte units, 16-byte aligned — or a dense copy
Tensor operand(const Tensor& t, int64_t* strides) {
    for (int i = 0; i < 3; ++i) strides[i] = t.size(i) > 1 ? t.stride(i) : 0;
    if (t.stride(3) == 1 && ((strides[0] | strides[1] | strides[2]) & 7) == 0 && strides[1] <= (1 << 23) && (uintptr_t)t.data_ptr() % 16 == 0) return t;
    const Tensor c = t.clone(c10::MemoryFormat::Contiguous);
    for (int i = 0; i < 3; ++i) strides[i] = c.stride(i);
    return c;
}

struct Attention : torch::autograd::Function<Attention> {
    struct Masks {
        Tensor prefix, documents, key_documents, lengths, slopes;
        double scale, softcap;
        bool causal;
    };
    // one call of the library; the operands' dense copies live until the work is enqueued
    static void call(const Tensor& q, const Tensor& k, const Tensor& v, const Masks& m, const Tensor& out, const Tensor& rest, const Tensor& lse, const Tensor& dout, const Tensor& dq,
                     const Tensor& dk, const Tensor& dv, n3d_stream_t stream) {
        n3d_attention_desc d = {};
        const Tensor q_ = operand(q, d.q_strides), k_ = operand(k, d.k_strides), v_ = operand(v, d.v_strides);
        const Tensor do_ = dout.defined() ? operand(dout, d.dout_strides) : Tensor();
        d.q = q_.data_ptr();
        d.k = k_.data_ptr();
        d.v = v_.data_ptr();
        d.out = out.data_ptr();
        d.out_rest = ptr(rest);
        d.lse = (float*)ptr(lse);
        d.prefix = (const int*)ptr(m.prefix);
        d.lengths = (const int*)ptr(m.lengths);
        d.slopes = (const float*)ptr(m.slopes);
        if (m.documents.defined()) {
            d.q_documents = (const int*)ptr(m.documents);
            d.k_documents = (const int*)ptr(m.key_documents);
            d.q_doc_stride = m.documents.stride(0);
            d.k_doc_stride = m.key_documents.stride(0);
        }
        d.dout = ptr(do_);
        d.dq = ptr(dq);
        d.dk = ptr(dk);
        d.dv = ptr(dv);
        d.scale = (float)m.scale;
        d.softcap = (float)m.softcap;
        d.B = (int)q.size(0);
        d.Lq = (int)q.size(1);
        d.Lk = (int)k.size(1);
        d.heads_q = (int)q.size(2);
        d.heads_k = (int)k.size(2);
        d.D = (int)q.size(3);
        d.dtype = code(q);
        d.causal = m.causal;
        d.workspace_bytes = dout.defined() ? lib.attention_bwd_workspace(&d) : lib.attention_workspace(&d);
        check(d.workspace_bytes);
        Tensor ws;
        if (d.workspace_bytes) {
            ws = at::empty({d.workspace_bytes}, q.options().dtype(at::kByte));
            d.workspace = ws.data_ptr();
        }
        check(dout.defined() ? lib.attention_bwd(&d, stream) : lib.attention(&d, stream));
    }
    // out, lse, and (for a gradient) what rounding out left over
    static std::tuple<Tensor, Tensor, Tensor> run(const Tensor& q, const Tensor& k, const Tensor& v, const Masks& m, bool want_lse, bool want_rest) {
        Scope scope(q);
        const Tensor out = dense(q), none;
        const Tensor lse = want_lse ? at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat)) : Tensor();
        const Tensor rest = want_rest ? dense(q) : Tensor();
        if (q.numel()) call(q, k, v, m, out, rest, lse, none, none, none, none, scope.stream);
        return {out, lse, rest};
    }
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Masks& m) {
        const auto [out, lse, rest] = run(q, k, v, m, true, true);
        ctx->save_for_backward({q, k, v, out, lse, rest, m.prefix, m.documents, m.key_documents, m.lengths, m.slopes});
        ctx->saved_data["scale"] = m.scale;
        ctx->saved_data["softcap"] = m.softcap;
        ctx->saved_data["causal"] = m.causal;
        ctx->mark_non_differentiable({lse});
        ctx->set_materialize_grads(false);
        return {out, lse};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2];
        Tensor dq, dk, dv;
        if (grads[0].defined()) {
            const Masks m = {s[6], s[7], s[8], s[9], s[10], ctx->saved_data["scale"].toDouble(), ctx->saved_data["softcap"].toDouble(), ctx->saved_data["causal"].toBool()};
            const bool want_k = ctx->needs_input_grad(1), want_v = ctx->needs_input_grad(2);
            Scope scope(q);
            if (ctx->needs_input_grad(0)) dq = dense(q);
            if (want_k || want_v) {
                dk = dense(k);
                dv = dense(v);
            }
            if (q.numel()) {
                call(q, k, v, m, s[3], s[5], s[4], grads[0].resolve_neg(), dq, dk, dv, scope.stream);
            } else if (dk.defined()) {                                            // no queries: nothing flows
                dk.zero_();
                dv.zero_();
            }
            if (!want_k) dk = Tensor();
            if (!want_v) dv = Tensor();
        }
        return once({dq, dk, dv, Tensor()}, "attention");
    }
};

std::tuple<Tensor, Opt> attention(const Tensor& q, const Tensor& k, const Tensor& v, double scale, bool causal, const Opt& prefix, const Opt& documents,
                                  const Opt& key_documents, const Opt& lengths, double softcap, const Opt& slopes, bool want_lse) {
    const Attention::Masks m = {get(prefix), get(documents), get(key_documents), get(lengths), get(slopes), scale, softcap, causal};
    refuse("attention", {&q, &k, &v, &m.prefix, &m.documents, &m.key_documents, &m.lengths, &m.slopes});
    if (wants_grad({&q, &k, &v})) {
        variable_list r = Attention::apply(q, k, v, m);
        return {r[0], r[1]};
    }
    auto [out, lse, rest] = Attention::run(q, k, v, m, want_lse, false);
    return {out, lse.defined() ? Opt(lse) : Opt()};
}

}  // namespace

PYBIND11_MODULE(_token_ext, m) {
    m.attr("torch_version") = N3D_TORCH;                    // of the headers that this was compiled against
    m.def("bind", &bind);
    m.def("layer_norm", &layer_norm);
    m.def("rotary", &rotary);
    m.def("attention", &attention);
}
