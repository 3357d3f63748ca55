// mgx_policy_torch.cpp -- include/mgx_policy.h's calls for torch tensors: argument checks, outputs, autograd.  Host code only; the module
// magical_amd._policy_torch (magical_amd/policy.py is its public face).
//
// Why not from Python through ctypes, as the engine is called: these calls take microseconds on the GPU, and there is one per env-step.
// Measured on a batch of 64 x 18 scores, the host's time per call: forward 14 us from Python; forward and backward 120 us, of which the
// backward pass's own thread taking the interpreter, and the interpreter's work there, were 75 (torch's own product and its gradient: 49).
#include <ATen/ExpandUtils.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <unordered_set>
#include <vector>

#include "../../../include/mgx_policy.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// the loaded library's entry points (magical_amd/_native.py loads it; set by bind())
struct {
    decltype(&mgx_policy_last_error) last_error;
    decltype(&mgx_policy_workspace_bytes) workspace_bytes;
    decltype(&mgx_policy_stats_bytes) stats_bytes;
    decltype(&mgx_policy_log_probs) log_probs;
    decltype(&mgx_policy_log_probs_backward) log_probs_backward;
    decltype(&mgx_policy_sample) sample;
} C;
PyObject *mgx_error_type = nullptr;

struct MgxError : torch::PyTorchError {       // raised as magical_amd._native.MgxError
    explicit MgxError(const std::string &m) : torch::PyTorchError(m) {}
    PyObject *python_type() override { return mgx_error_type; }
};
void check(int rc) {
    if (rc < 0) throw MgxError("mgx error " + std::to_string(rc) + ": " + C.last_error());
}

// A tangent would not come out at the other end, and nobody would know: refused.  (Without tangents in the process: one look at a pointer.)
void refuse_tangent(const Tensor &t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t.defined() || !t._fw_grad(0).defined(),
                                "action_log_probs has no forward-mode derivative");
}
// In torch.jit.trace the results would become constants.
void refuse_tracing() { TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing(), "the operators on action scores cannot be traced"); }

// what lies in memory behind a tensor is its values (no negation put off, no zeros without memory)
Tensor plain(const Tensor &t) { return t._is_zerotensor() ? t.clone() : t.is_neg() ? t.resolve_neg() : t; }

// rows x n scores as the C calls take them, and the tensors behind the pointers
struct Scores {
    int dtype;
    Tensor x, mask;
    int64_t rows, n, stride, mask_stride = 0;
    const uint8_t *mask_ptr = nullptr;
    double temperature;

    Scores(const Tensor &logits, const OptTensor &m, double temperature_) : temperature(temperature_) {
        switch (logits.scalar_type()) {
            case at::kFloat: dtype = MGX_REAL_F32; break;
            case at::kHalf: dtype = MGX_REAL_F16; break;
            case at::kBFloat16: dtype = MGX_REAL_BF16; break;
            default: TORCH_CHECK_TYPE(false, "logits: float32, float16 or bfloat16, got ", logits.scalar_type());
        }
        TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1, "logits: [..., n] with n >= 1, got ", logits.sizes());
        TORCH_CHECK_VALUE(temperature >= 1e-37 && temperature <= 1e37, "temperature: 1e-37 ... 1e37, got ", temperature);
        n = logits.size(-1);
        x = dense_rows(logits);
        rows = x.size(0);
        stride = x.stride(0);
        if (!m) return;
        TORCH_CHECK_TYPE(m->scalar_type() == at::kBool, "mask: a bool tensor, got ", m->scalar_type());
        TORCH_CHECK_VALUE(m->device() == logits.device(), "mask is on ", m->device(), ", logits on ", logits.device());
        TORCH_CHECK_VALUE(at::is_expandable_to(m->sizes(), logits.sizes()), "mask ", m->sizes(), " does not broadcast to logits ", logits.sizes());
        mask = dense_rows(m->expand(logits.sizes()));
        mask_ptr = (const uint8_t *)mask.data_ptr();
        mask_stride = mask.stride(0);
    }
    // [rows][n] with neighbouring columns: a view where there is one
    Tensor dense_rows(const Tensor &t) const {
        const Tensor p = plain(t), v = p.dim() == 2 ? p : p.reshape({p.numel() / n, n});
        return n > 1 && v.stride(1) != 1 ? v.contiguous() : v;
    }
};
#define SCORES(s) (s).dtype, (s).x.data_ptr(), (s).rows, (s).n, (s).stride, (s).mask_ptr, (s).mask_stride, (s).temperature

void *stream_of(const Tensor &t) {
    if (!t.is_cuda()) throw MgxError("magical_amd runs on an MI355X (torch device \"cuda:N\"); there is no CPU fallback");
    return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

Tensor workspace(int op, const Scores &s, int64_t top, const Tensor &like) {
    const int64_t bytes = C.workspace_bytes(op, s.dtype, s.rows, s.n, (int)top);
    return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}

struct Forward {
    Tensor log_prob, entropy, top_log_probs, top_actions, stats, actions;
};

Forward forward(const Tensor &logits, const Tensor &actions, const OptTensor &mask, double temperature, int64_t top, bool for_backward) {
    const Scores s(logits, mask, temperature);
    const at::IntArrayRef lead = logits.sizes().slice(0, logits.dim() - 1);
    TORCH_CHECK_TYPE(actions.scalar_type() == at::kInt || actions.scalar_type() == at::kLong, "actions: an int32 or int64 tensor, got ",
                     actions.scalar_type());
    TORCH_CHECK_VALUE(actions.device() == logits.device(), "actions are on ", actions.device(), ", logits on ", logits.device());
    TORCH_CHECK_VALUE(actions.sizes() == lead, "actions: one for each row of logits, ", lead, ", got ", actions.sizes());
    TORCH_CHECK_VALUE(top >= 0 && top <= MGX_POLICY_MAX_TOP && top <= s.n, "top: 0 ... min(n, ", (int)MGX_POLICY_MAX_TOP, "), got ", top,
                      " for n = ", s.n);
    void *stream = stream_of(logits);
    const at::TensorOptions f32 = logits.options().dtype(at::kFloat);
    Forward f;
    f.actions = plain(actions).contiguous();
    f.log_prob = at::empty(lead, f32);
    f.entropy = at::empty(lead, f32);
    if (for_backward)
        if (const int64_t bytes = C.stats_bytes(s.rows, s.n)) f.stats = at::empty({bytes / 4}, f32);
    if (top) {
        at::DimVector shape(lead.begin(), lead.end());
        shape.push_back(top);
        f.top_log_probs = at::empty(shape, f32);
        f.top_actions = at::empty(shape, f32.dtype(at::kInt));
    }
    const Tensor ws = workspace(MGX_POLICY_LOG_PROBS, s, top, logits);
    check(C.log_probs(logits.device().index(), SCORES(s), f.actions.data_ptr(), (int)f.actions.element_size(), (int)top,
                      f.log_prob.data_ptr<float>(), f.entropy.data_ptr<float>(), f.stats.defined() ? f.stats.data_ptr<float>() : nullptr,
                      top ? f.top_log_probs.data_ptr<float>() : nullptr, top ? f.top_actions.data_ptr<int32_t>() : nullptr,
                      ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? ws.numel() : 0, stream));
    return f;
}

// an upstream gradient, one f32 a row: (pointer, row stride), stride 0 for an expanded scalar's
struct Upstream {
    Tensor g;
    const float *ptr = nullptr;
    int64_t stride = 0;
    explicit Upstream(const Tensor &t) {
        if (!t.defined()) return;
        g = plain(t);
        if (g.dim() != 1) g = g.reshape({-1});
        ptr = g.const_data_ptr<float>();
        stride = g.stride(0);
    }
};

// A gradient arrives on the stream of the forward call that it belongs to, a leaf's on that on which an earlier call first asked for it, as long as
// results of such calls are alive.  A captured backward pass would have to wait for that stream, and the default stream cannot take part in a
// capture: torch ends the process.  Refused before: where the logits are such a leaf by the captured forward call, else (a network's weights) by the
// backward pass, as soon as it gets here, for whatever it is going to reach behind this node.
bool capturing(c10::Device device) {
    const c10::DeviceGuard guard(device);
    return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
}
bool on_default_stream(torch::autograd::Node &node) {
    const auto stream = node.stream();
    return stream && stream->id() == c10::hip::getDefaultHIPStream(stream->device_index()).id();
}
void refuse_captured_backward_beside_eager_graph(const torch::autograd::Node &node, c10::Device device) {
    if (!capturing(device)) return;
    const auto *reached = torch::autograd::get_current_graph_task_exec_info();          // (none or empty: every node)
    std::unordered_set<const torch::autograd::Node *> seen;
    std::vector<const torch::autograd::Node *> left{&node};
    while (!left.empty()) {
        const auto *from = left.back();
        left.pop_back();
        for (const torch::autograd::Edge &edge : from->next_edges()) {
            torch::autograd::Node *const to = edge.function.get();
            if (!to || !seen.insert(to).second) continue;
            if (reached && !reached->empty()) {
                const auto it = reached->find(to);
                if (it == reached->end() || !it->second.should_execute()) continue;
            }
            if (on_default_stream(*to))
                throw MgxError("something behind the logits (a network's weight, the logits themselves) still belongs to results of earlier calls on the "
                               "default stream: free these results before the forward and the backward pass are captured, both of them");
            left.push_back(to);
        }
    }
}
void refuse_capture_beside_eager_graph(const Tensor &logits) {
    if (!logits.is_leaf() || !logits.is_cuda()) return;
    const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(logits);
    if (accumulator && on_default_stream(*accumulator) && capturing(logits.device()))
        throw MgxError("logits that need a gradient still belong to results of earlier calls on the default stream: free these results before this "
                       "call is captured, or give logits.detach()");
}

// The backward pass's node.  (A custom Function keeps the same, with a dictionary and checks that cost 2 us a call.)
struct LogProbsBackward : torch::autograd::Node {
    SavedVariable logits, actions, mask, stats, entropy;
    double temperature = 1;

    variable_list apply(variable_list &&grads) override {
        variable_list out(1);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        refuse_tangent(grads[0]);
        refuse_tangent(grads[1]);
        refuse_captured_backward_beside_eager_graph(*this, (grads[0].defined() ? grads[0] : grads[1]).device());
        std::lock_guard<std::mutex> lock(mutex_);
        const Tensor x = logits.unpack(), a = actions.unpack(), m = mask.unpack(), st = stats.unpack(), h = entropy.unpack(shared_from_this());
        const bool differentiated = at::GradMode::is_enabled();
        at::NoGradGuard no_grad;
        const Scores s(x, m.defined() ? OptTensor(m) : OptTensor(), temperature);
        const Upstream g_lp(grads[0]), g_h(grads[1]);
        Tensor grad = at::empty(x.sizes(), x.options());
        check(C.log_probs_backward(x.device().index(), SCORES(s), a.data_ptr(), (int)a.element_size(),
                                   st.defined() ? st.const_data_ptr<float>() : nullptr, h.const_data_ptr<float>(), g_lp.ptr, g_lp.stride, g_h.ptr,
                                   g_h.stride, grad.data_ptr(), stream_of(x)));
        if (differentiated) {      // create_graph: the gradient has none of its own, and says so when it is asked for
            at::AutoGradMode with_grad(true);
            Tensor fake = grad.detach();
            fake.set_requires_grad(true);
            auto refuse = std::make_shared<torch::autograd::DelayedError>("action_log_probs is differentiable once", 1);
            grad = (*refuse)({fake})[0];
        }
        out[0] = grad;
        return out;
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable *v : {&logits, &actions, &mask, &stats, &entropy}) v->reset_data();
    }
    std::string name() const override { return "ActionLogProbsBackward"; }
};

Forward forward_with_graph(const Tensor &logits, const Tensor &actions, const OptTensor &mask, double temperature, int64_t top) {
    Forward f;
    refuse_capture_beside_eager_graph(logits);
    {
        at::NoGradGuard no_grad;
        f = forward(logits, actions, mask, temperature, top, true);
    }
    std::shared_ptr<LogProbsBackward> node(new LogProbsBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    node->temperature = temperature;
    node->logits = SavedVariable(logits, false);
    node->actions = SavedVariable(f.actions, false);
    if (mask) node->mask = SavedVariable(*mask, false);
    if (f.stats.defined()) node->stats = SavedVariable(f.stats, false);
    torch::autograd::set_history(f.log_prob, node);
    torch::autograd::set_history(f.entropy, node);
    node->entropy = SavedVariable(f.entropy, true);
    return f;
}

py::object or_none(const Tensor &t) { return t.defined() ? py::cast(t) : py::none(); }

py::tuple log_probs(const Tensor &logits, const Tensor &actions, const OptTensor &mask, double temperature, int64_t top) {
    refuse_tangent(logits);
    refuse_tracing();
    const Forward f = at::GradMode::is_enabled() && logits.requires_grad() ? forward_with_graph(logits, actions, mask, temperature, top)
                                                                           : forward(logits, actions, mask, temperature, top, false);
    return py::make_tuple(f.log_prob, f.entropy, or_none(f.top_log_probs), or_none(f.top_actions));
}

py::tuple sample(const Tensor &logits, const Tensor &uniforms, const OptTensor &mask, double temperature) {
    refuse_tracing();
    const Scores s(logits, mask, temperature);
    const at::IntArrayRef lead = logits.sizes().slice(0, logits.dim() - 1);
    TORCH_CHECK_TYPE(uniforms.scalar_type() == at::kFloat || uniforms.scalar_type() == at::kDouble,
                     "uniforms: a float32 or float64 tensor, got ", uniforms.scalar_type());
    TORCH_CHECK_VALUE(uniforms.device() == logits.device(), "uniforms are on ", uniforms.device(), ", logits on ", logits.device());
    TORCH_CHECK_VALUE(uniforms.sizes() == lead, "uniforms: one for each row of logits, ", lead, ", got ", uniforms.sizes());
    void *stream = stream_of(logits);
    const at::TensorOptions f32 = logits.options().dtype(at::kFloat);
    const Tensor u = plain(uniforms).contiguous(), action = at::empty(lead, f32.dtype(at::kInt)), log_prob = at::empty(lead, f32),
                 entropy = at::empty(lead, f32), ws = workspace(MGX_POLICY_SAMPLE, s, 0, logits);
    check(C.sample(logits.device().index(), SCORES(s), u.data_ptr(), (int)u.element_size(), action.data_ptr<int32_t>(),
                   log_prob.data_ptr<float>(), entropy.data_ptr<float>(), ws.defined() ? ws.data_ptr() : nullptr,
                   ws.defined() ? ws.numel() : 0, stream));
    return py::make_tuple(action, log_prob, entropy);
}

void bind(const py::dict &entries, const py::object &error_type) {
    const auto address = [&](const char *name) { return (void *)entries[name].cast<uintptr_t>(); };
    C.last_error = (decltype(C.last_error))address("mgx_policy_last_error");
    C.workspace_bytes = (decltype(C.workspace_bytes))address("mgx_policy_workspace_bytes");
    C.stats_bytes = (decltype(C.stats_bytes))address("mgx_policy_stats_bytes");
    C.log_probs = (decltype(C.log_probs))address("mgx_policy_log_probs");
    C.log_probs_backward = (decltype(C.log_probs_backward))address("mgx_policy_log_probs_backward");
    C.sample = (decltype(C.sample))address("mgx_policy_sample");
    mgx_error_type = error_type.inc_ref().ptr();
}

}  // namespace

PYBIND11_MODULE(_policy_torch, m) {
    m.def("bind", &bind);
    m.def("log_probs", torch::wrap_pybind_function(log_probs));
    m.def("sample", torch::wrap_pybind_function(sample));
}
