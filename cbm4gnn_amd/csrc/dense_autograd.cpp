// The differentiable calls of the dense operators as torch sees them: allocation of outputs and workspaces, the launches
// of libcbm_hip, and the autograd nodes.  Argument checks are the Python callers'.
//
// Compiled, because a training step on a small graph is bound by the host: autograd runs a backward on a thread of its
// own, and a node written in Python makes that thread take turns with the caller for the interpreter.  Forward and
// backward of 232 965 x 41 labels take 26 us of kernels; issuing them takes 47 us, 96 with nodes in Python (on the same
// kind of host an empty Python node takes 41); of a norm of 24 001 x 602 in 37 graphs 83 us, 147 in Python; scores
// without a gradient 9 us, 16 in Python.
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <optional>
#include <tuple>

#include "../../include/cbm_hip.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

// What the Python bindings raise for the same status.
void check(int rc, const char* where) {
    TORCH_CHECK_VALUE(rc != CBM_ERR_NULL && rc != CBM_ERR_SHAPE, where, ": ", cbm_status_string(rc), " (status ", rc, ")");
    TORCH_CHECK(rc == CBM_OK, where, ": ", cbm_status_string(rc), " (status ", rc, ")");
}

int dtype_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return CBM_DTYPE_F32;
        case at::kBFloat16: return CBM_DTYPE_BF16;
        case at::kHalf: return CBM_DTYPE_F16;
        default: TORCH_CHECK(false, "unsupported element type ", t.scalar_type());
    }
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

template <typename T>
T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
template <typename T>
T* ptr(const MaybeTensor& t) { return t ? ptr<T>(*t) : nullptr; }

Tensor floats(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(at::kFloat)); }
Tensor workspace(int64_t n, const Tensor& like) { return n > 0 ? floats({n}, like) : Tensor(); }

// t as rows of `width` values, unit stride along them; rows whose stride does not allow it are copied.
Tensor rows_of(Tensor t, int64_t width) {
    if (t.dim() != 2) t = t.reshape({-1, width});
    if ((width > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < width)) t = t.contiguous();
    return t;
}
int64_t ld(const Tensor& m) { return m.size(0) > 1 ? m.stride(0) : std::max<int64_t>(m.size(1), 1); }

// Refuses what would go on with a wrong result, for the kernels write through raw pointers, unseen by torch:
//   * forward mode: a result without a tangent would be read as a derivative of zero;
//   * a tracer (torch.jit.trace, make_fx): of a call it would record the allocation of the result, and nothing that fills it.
void not_followed(at::ArrayRef<MaybeTensor> inputs, const char* where) {
    using c10::impl::TorchDispatchModeKey;
    using c10::impl::TorchDispatchModeTLS;
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() && !TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY), where,
                                " cannot be traced: a tracer does not see what its kernels write");
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const MaybeTensor& t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t || !t->defined() || !t->_fw_grad(0).defined(), where,
                                    " has no forward-mode derivative; torch.autograd differentiates it in reverse mode");
}

// Gradients have no derivative of their own: where a graph of them is asked for, following it is an error.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list wanted;
    for (Tensor& g : grads)
        if (g.defined()) wanted.push_back(g.detach().requires_grad_(true));
    auto refuse = std::make_shared<torch::autograd::DelayedError>("the gradient of this operator cannot be differentiated again",
                                                                  static_cast<int64_t>(wanted.size()));
    const variable_list refusing = (*refuse)(std::move(wanted));
    size_t k = 0;
    for (Tensor& g : grads)
        if (g.defined()) g = refusing[k++];
    return grads;
}

// ---------------------------------------------------------------------------------------------
// label scores
// ---------------------------------------------------------------------------------------------
struct Scores { Tensor logp, entropy, top_logp, top_index, stats; };

Scores run_scores(const Tensor& z, const MaybeTensor& labels, bool entropy, int64_t top, int64_t ignore_index, bool keep) {
    const c10::DeviceGuard guard(z.device());
    const int64_t rows = z.size(0), classes = z.size(1);
    const int dt = dtype_of(z);
    Scores s;
    if (labels) s.logp = floats({rows}, z);
    if (entropy) s.entropy = floats({rows}, z);
    if (top) {
        s.top_logp = floats({rows, top}, z);
        s.top_index = at::empty({rows, top}, z.options().dtype(at::kLong));
    }
    if (keep) s.stats = floats({rows, 2}, z);
    const Tensor ws = workspace(cbm_label_scores_workspace_floats(rows, classes, top, dt), z);
    check(cbm_label_scores(z.data_ptr(), ptr<int64_t>(labels), ptr<float>(s.logp), ptr<float>(s.entropy), ptr<float>(s.top_logp),
                           ptr<int64_t>(s.top_index), ptr<float>(s.stats), ptr<float>(ws), rows, classes, top, ld(z), ignore_index, dt,
                           stream_of(z)),
          "cbm_label_scores");
    return s;
}

struct LabelScores : torch::autograd::Function<LabelScores> {
    static variable_list forward(AutogradContext* ctx, const Tensor& z, const MaybeTensor& labels, bool entropy, int64_t top,
                                 int64_t ignore_index) {
        const Scores s = run_scores(z, labels, entropy, top, ignore_index, true);
        ctx->save_for_backward({z, labels ? *labels : Tensor(), s.stats, s.entropy, s.top_index});
        ctx->saved_data["top"] = top;
        ctx->saved_data["ignore"] = ignore_index;
        ctx->set_materialize_grads(false);
        if (top) ctx->mark_non_differentiable({s.top_index});
        variable_list out;
        for (const Tensor& t : {s.logp, s.entropy, s.top_logp, s.top_index})
            if (t.defined()) out.push_back(t);
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &z = saved[0], &labels = saved[1], &stats = saved[2], &entropy = saved[3], &top_index = saved[4];
        const int64_t top = ctx->saved_data["top"].toInt(), ignore_index = ctx->saved_data["ignore"].toInt();
        const c10::DeviceGuard guard(z.device());
        size_t k = 0;
        auto next = [&](bool there) {                       // gradients come in the order of the outputs that there are
            Tensor g = there ? grads[k++] : Tensor();
            return g.defined() ? g.contiguous() : g;
        };
        const Tensor g_logp = next(labels.defined()), g_entropy = next(entropy.defined()), g_top = next(top > 0);
        const int64_t rows = z.size(0), classes = z.size(1);
        Tensor grad = at::empty({rows, classes}, z.options());
        check(cbm_label_scores_backward(z.data_ptr(), ptr<int64_t>(labels), ptr<float>(stats), ptr<float>(entropy), ptr<int64_t>(top_index),
                                        ptr<float>(g_logp), ptr<float>(g_entropy), ptr<float>(g_top), grad.data_ptr(), rows, classes, top,
                                        ld(z), classes, ignore_index, dtype_of(z), stream_of(z)),
              "cbm_label_scores_backward");
        return once({grad, Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

std::tuple<MaybeTensor, MaybeTensor, MaybeTensor, MaybeTensor> label_scores(const Tensor& z, const MaybeTensor& labels, bool entropy,
                                                                            int64_t top, int64_t ignore_index) {
    not_followed({z}, "label_log_probs");
    auto some = [](const Tensor& t) { return t.defined() ? MaybeTensor(t) : std::nullopt; };
    if (!at::GradMode::is_enabled() || !z.requires_grad()) {
        const Scores s = run_scores(z, labels, entropy, top, ignore_index, false);
        return {some(s.logp), some(s.entropy), some(s.top_logp), some(s.top_index)};
    }
    const variable_list out = LabelScores::apply(z, labels, entropy, top, ignore_index);
    size_t k = 0;
    auto next = [&](bool there) { return there ? MaybeTensor(out[k++]) : std::nullopt; };
    MaybeTensor logp = next(labels.has_value()), ent = next(entropy), top_logp = next(top > 0), top_index = next(top > 0);
    return {logp, ent, top_logp, top_index};
}

// ---------------------------------------------------------------------------------------------
// group norm
// ---------------------------------------------------------------------------------------------
// The rows of a batch of graphs, with the device arrays that its kernels index with: a node that holds the batch holds them.
struct NormBatch : torch::CustomClassHolder {
    cbm_norm_batch rows{};
    variable_list arrays;                  // none (equal lengths), or ptr, pieces, piece_ptr, order (int32)

    NormBatch(int64_t samples, int64_t max_len, int64_t n, int64_t piece_rows, int64_t n_pieces, variable_list held)
        : arrays(std::move(held)) {
        rows.samples = samples; rows.max_len = max_len; rows.rows = n; rows.piece_rows = piece_rows; rows.n_pieces = n_pieces;
        if (!arrays.empty()) {
            rows.ptr = ptr<int32_t>(arrays.at(0));
            rows.pieces = ptr<int32_t>(arrays.at(1));
            rows.piece_ptr = ptr<int32_t>(arrays.at(2));
            rows.order = ptr<int32_t>(arrays.at(3));
        }
    }
};
using Batch = c10::intrusive_ptr<NormBatch>;

struct Normed { Tensor y, mean, rstd; };

Normed run_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, const cbm_norm_batch& B, int64_t groups, double eps,
                int64_t act, bool keep) {
    const c10::DeviceGuard guard(x.device());
    const Tensor m = rows_of(x, x.size(-1));
    const int64_t ch = m.size(1);
    const int dt = dtype_of(x);
    Normed n;
    n.y = at::empty(x.sizes(), x.options());
    if (keep) {
        n.mean = floats({B.samples, groups}, x);
        n.rstd = floats({B.samples, groups}, x);
    }
    const Tensor ws = workspace(cbm_group_norm_workspace_floats(&B, ch, groups, dt, 0), x);
    check(cbm_group_norm_forward(&B, m.data_ptr(), n.y.data_ptr(), ptr<float>(weight), ptr<float>(bias), ptr<float>(n.mean),
                                 ptr<float>(n.rstd), ptr<float>(ws), ch, groups, ld(m), ch, eps, act, dt, stream_of(x)),
          "cbm_group_norm_forward");
    return n;
}

struct GroupNorm : torch::autograd::Function<GroupNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, const Batch& batch,
                          int64_t groups, double eps, int64_t act) {
        const Normed n = run_norm(x, weight, bias, batch->rows, groups, eps, act, true);
        ctx->save_for_backward({x, weight ? *weight : Tensor(), bias ? *bias : Tensor(), n.mean, n.rstd});
        ctx->saved_data["batch"] = c10::IValue::make_capsule(batch);
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["act"] = act;
        return n.y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2];
        const Batch batch = c10::static_intrusive_pointer_cast<NormBatch>(ctx->saved_data["batch"].toCapsule());
        const int64_t groups = ctx->saved_data["groups"].toInt(), act = ctx->saved_data["act"].toInt();
        const c10::DeviceGuard guard(x.device());
        const Tensor m = rows_of(x, x.size(-1)), g = rows_of(grads[0], x.size(-1));
        const int64_t ch = m.size(1);
        const int dt = dtype_of(x);
        size_t edge = 0;                                    // counts the tensors among the arguments
        const bool need_x = ctx->needs_input_grad(edge++);
        const bool need_w = weight.defined() && ctx->needs_input_grad(edge++);
        const bool need_b = bias.defined() && ctx->needs_input_grad(edge++);
        Tensor dx = need_x ? at::empty(x.sizes(), x.options()) : Tensor();
        Tensor dw = need_w ? floats({ch}, x) : Tensor(), db = need_b ? floats({ch}, x) : Tensor();
        const Tensor ws = workspace(cbm_group_norm_workspace_floats(&batch->rows, ch, groups, dt, 1), x);
        check(cbm_group_norm_backward(&batch->rows, m.data_ptr(), g.data_ptr(), ptr<void>(dx), ptr<float>(weight), ptr<float>(bias),
                                      ptr<float>(saved[3]), ptr<float>(saved[4]), ptr<float>(dw), ptr<float>(db), ptr<float>(ws), ch,
                                      groups, ld(m), ld(g), ch, act, dt, stream_of(x)),
              "cbm_group_norm_backward");
        return once({dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

Tensor group_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, const Batch& batch, int64_t groups, double eps,
                  int64_t act) {
    not_followed({x, weight, bias}, "group_norm");
    auto grad = [](const MaybeTensor& t) { return t && t->requires_grad(); };
    if (!at::GradMode::is_enabled() || !(x.requires_grad() || grad(weight) || grad(bias)))
        return run_norm(x, weight, bias, batch->rows, groups, eps, act, false).y;
    return GroupNorm::apply(x, weight, bias, batch, groups, eps, act);
}

}  // namespace

PYBIND11_MODULE(cbm_autograd, m) {
    const auto unlocked = py::call_guard<py::gil_scoped_release>();
    m.def("label_scores", &label_scores, unlocked);
    m.def("group_norm", &group_norm, unlocked);
    m.def("not_followed", [](const std::vector<Tensor>& inputs, const std::string& where) {
        not_followed(std::vector<MaybeTensor>(inputs.begin(), inputs.end()), where.c_str());
    });
    py::class_<NormBatch, Batch>(m, "NormBatch")
        .def(py::init<int64_t, int64_t, int64_t, int64_t, int64_t, variable_list>())
        .def_readonly("arrays", &NormBatch::arrays);
}
