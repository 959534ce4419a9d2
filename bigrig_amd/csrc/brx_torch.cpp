// The calls of norm.py that record a gradient, and their gradients, as nodes of torch's graph in C++.
//
// torch runs gradients on a thread of its own. A node written in Python takes the interpreter there while the thread that waits
// for it gives it up, and both run cold: of a short pass (some hundred rows) that is most of the time. Here a gradient is its
// allocations and its launches. Arguments come checked from norm.py, the work is libbrx's (brx_norm_forward, brx_norm_backward).
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include "brx.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

void check(int rc) { TORCH_CHECK(rc == BRX_OK, "libbrx error ", rc, ": ", brx_last_error()); }

int type_of(const Tensor& t) {
    if (!t.defined()) return 0;
    return t.scalar_type() == at::kBFloat16 ? BRX_DT_BF16 : t.scalar_type() == at::kHalf ? BRX_DT_F16 : BRX_DT_F32;
}
const void* from(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* to(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
float* floats(const Tensor& t) { return t.defined() ? t.mutable_data_ptr<float>() : nullptr; }
int64_t row_of(const Tensor& t) { return !t.defined() ? 0 : t.size(0) > 1 ? t.stride(0) : t.size(1); }
void* stream_on(at::Device device) { return c10::hip::getCurrentHIPStream(device.index()).stream(); }
Tensor or_none(const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); }

constexpr int kGateChannel = 1;             // (a gate form, brx.h)

struct NormBackward : torch::autograd::Node {
    enum { kY, kR, kPost, kGate, kNext, kInputs };      // the edges
    SavedVariable y, r, post, gate, next;   // r: what h was made of
    Tensor rstd_y, rstd_n;
    at::TensorOptions r_options;
    at::ScalarType h_type = at::kFloat;
    double scale = 1.0;
    int form = 0, T = 0, H = 0;
    bool leave = false, makes_h = false;    // outputs: new (of leave) and h

    std::string name() const override { return "BlockNormBackward"; }

    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable* v : {&y, &r, &post, &gate, &next}) v->reset_data();
        rstd_y.reset();
        rstd_n.reset();
    }

    variable_list apply(variable_list&& grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        TORCH_CHECK(!at::GradMode::is_enabled(), "this gradient is taken once: create_graph=True is refused");
        for (const Tensor& g : grads) refuse_tangent(g);
        variable_list got(kInputs);
        Tensor d_new, d_h;
        if (leave) d_new = grads[0];
        if (makes_h) d_h = grads[leave ? 1 : 0];
        if (!leave && !d_h.defined()) d_h = at::zeros({T, H}, r_options.dtype(h_type));
        if (!d_new.defined() && !d_h.defined()) return got;
        if (d_new.defined()) d_new = d_new.contiguous();
        if (d_h.defined()) d_h = d_h.contiguous();
        const Tensor y_ = y.unpack(), r_ = r.unpack(leave ? shared_from_this() : nullptr), post_ = post.unpack(), gate_ = gate.unpack(),
                     next_ = next.unpack();
        auto rows = [&](const at::TensorOptions& o) { return at::empty({T, H}, o); };
        auto whole = [&](const Tensor& t) { return T ? at::empty_like(t) : at::zeros_like(t); };
        if (task_should_compute_output(kY)) got[kY] = rows(y_.options());
        // (without an h the residual's gradient is the one given)
        if (task_should_compute_output(kR)) got[kR] = makes_h ? rows(r_options) : d_new;
        if (task_should_compute_output(kPost)) got[kPost] = whole(post_);
        if (task_should_compute_output(kGate)) got[kGate] = whole(gate_);
        if (task_should_compute_output(kNext) && d_h.defined()) got[kNext] = whole(next_);
        if (!got[kY].defined() && !got[kPost].defined() && !got[kGate].defined() && !makes_h) return got;
        Tensor ws;
        size_t need = 0;
        if (got[kPost].defined() || got[kNext].defined() || (got[kGate].defined() && form == kGateChannel)) {
            check(brx_norm_workspace_bytes(T, H, &need));
            ws = at::empty({(int64_t)need}, r_options.dtype(at::kByte));
        }
        const int r_type = r_options.dtype() == at::kBFloat16 ? BRX_DT_BF16 : r_options.dtype() == at::kHalf ? BRX_DT_F16 : BRX_DT_F32;
        check(brx_norm_backward(from(y_), row_of(y_), leave ? type_of(y_) : type_of(d_h), from(r_), row_of(r_), r_type, from(post_),
                                type_of(post_), from(gate_), form, type_of(gate_), from(next_), type_of(next_), (float)scale, T, H,
                                floats(rstd_y), floats(rstd_n), from(d_new), from(d_h), to(got[kY]), makes_h ? to(got[kR]) : nullptr, to(got[kGate]),
                                to(got[kPost]), to(got[kNext]), to(ws), need, stream_on(r_options.device())));
        return got;
    }

    static void refuse_tangent(const Tensor& t) {
        TORCH_CHECK(!torch::autograd::isFwGradDefined(t), "a tensor with a tangent: there are no forward-mode derivatives");
    }
};

// (new, h): rows r [T, H] and, for leave, y [T, H].
std::tuple<Tensor, Tensor> norms(const Tensor& y, const Tensor& r, const Tensor& post, const Tensor& gate, int64_t form, const Tensor& next,
                                 double scale, double eps, bool makes_h, at::ScalarType h_type) {
    for (const Tensor* t : {&y, &r, &post, &gate, &next}) NormBackward::refuse_tangent(*t);
    const int T = (int)r.size(0), H = (int)r.size(1);
    Tensor fresh, h, rstd_y, rstd_n;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        if (y.defined()) fresh = at::empty({T, H}, r.options());
        if (makes_h) h = at::empty({T, H}, r.options().dtype(h_type));
        if (post.defined()) rstd_y = at::empty({T}, r.options().dtype(at::kFloat));
        if (makes_h) rstd_n = at::empty({T}, r.options().dtype(at::kFloat));
        check(brx_norm_forward(from(y), row_of(y), type_of(y.defined() ? y : h), from(r), row_of(r), type_of(r), from(post), type_of(post),
                               from(gate), (int)form, type_of(gate), from(next), type_of(next), (float)scale, (float)eps, T, H, to(fresh),
                               to(h), floats(rstd_y), floats(rstd_n), stream_on(r.device())));
    }
    if (torch::autograd::compute_requires_grad(y, r, post, gate, next)) {
        std::shared_ptr<NormBackward> node(new NormBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(y, r, post, gate, next));
        node->leave = y.defined();
        node->makes_h = makes_h;
        node->r_options = r.options();
        node->h_type = h_type;
        node->scale = scale;
        node->form = (int)form;
        node->T = T;
        node->H = H;
        node->rstd_y = rstd_y;
        node->rstd_n = rstd_n;
        if (fresh.defined()) torch::autograd::set_history(fresh, node);
        if (h.defined()) torch::autograd::set_history(h, node);
        node->y = SavedVariable(y, false);
        node->post = SavedVariable(post, false);
        node->gate = SavedVariable(gate, false);
        node->next = SavedVariable(next, false);
        if (makes_h) node->r = y.defined() ? SavedVariable(fresh, true) : SavedVariable(r, false);
    }
    return {fresh, h};
}

Tensor enter(const Tensor& x, const MaybeTensor& weight, double eps, at::ScalarType dtype) {
    return std::get<1>(norms(Tensor(), x, Tensor(), Tensor(), 0, or_none(weight), 1.0, eps, true, dtype));
}

Tensor leave(const Tensor& y, const Tensor& residual, const MaybeTensor& weight, const MaybeTensor& gate, int64_t form, double scale,
             double eps) {
    return std::get<0>(norms(y, residual, or_none(weight), or_none(gate), form, Tensor(), scale, eps, false, y.scalar_type()));
}

std::tuple<Tensor, Tensor> leave_enter(const Tensor& y, const Tensor& residual, const MaybeTensor& weight, const MaybeTensor& gate,
                                       int64_t form, double scale, const Tensor& next_weight, double eps) {
    return norms(y, residual, or_none(weight), or_none(gate), form, next_weight, scale, eps, true, y.scalar_type());
}

}  // namespace

TORCH_LIBRARY(brx, m) {
    m.def("enter(Tensor x, Tensor? weight, float eps, ScalarType dtype) -> Tensor", enter);
    m.def("leave(Tensor y, Tensor residual, Tensor? weight, Tensor? gate, int form, float scale, float eps) -> Tensor", leave);
    m.def("leave_enter(Tensor y, Tensor residual, Tensor? weight, Tensor? gate, int form, float scale, Tensor next_weight, float eps)"
          " -> (Tensor, Tensor)", leave_enter);
}
