// Autograd nodes of the losses on scores and gate logits (difflogic/losses.py checks their arguments and has their plain forms for CPU tensors).
#include "loss_nodes.h"

#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_cpp_function.h>

#include <mutex>

#include "convlogic_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

void check(int rc)
{
    TORCH_CHECK(rc == CLG_OK, clg_last_error());
}
void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
// the graph that the current stream is recorded into, 0 for none
int64_t recording()
{
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return 0;
    hipStreamCaptureStatus status;
    unsigned long long id = 0;
    C10_HIP_CHECK(hipStreamGetCaptureInfo(c10::hip::getCurrentHIPStream().stream(), &status, &id));
    return (int64_t)id + 1;
}
int code_of(const Tensor &t)
{
    switch (t.scalar_type()) {
    case at::kFloat: return CLG_F32;
    case at::kDouble: return CLG_F64;
    case at::kHalf: return CLG_F16;
    case at::kBFloat16: return CLG_BF16;
    default: TORCH_CHECK(false, "float32, float64, float16 or bfloat16 expected, got ", t.scalar_type());
    }
}
at::TensorOptions wide(const Tensor &t) { return t.options().dtype(t.scalar_type() == at::kDouble ? at::kDouble : at::kFloat); }

// [..., columns] as rows of dense columns
struct Rows {
    const void *at;
    int64_t rows, stride, cols;
    explicit Rows(const Tensor &t) : at(t.data_ptr()), cols(t.size(-1))
    {
        rows = t.numel() / cols;
        stride = t.is_contiguous() ? cols : t.stride(0);
    }
};
// t itself where Rows can say where its rows are
Tensor rows_of(const Tensor &t)
{
    if (t.is_contiguous() || (t.dim() == 2 && t.stride(1) == 1)) return t;
    return t.contiguous();
}

variable_list once(variable_list grads) { return once_only(std::move(grads), "the gradient of this loss cannot be differentiated"); }

// ---- top logits ------------------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor, Tensor> top_logits(const Tensor &logits_in, int64_t k, double temperature)
{
    const c10::OptionalDeviceGuard guard(logits_in.device());
    const Tensor logits = rows_of(logits_in.detach());
    const Rows r(logits);
    auto shape = logits.sizes().vec();
    shape.back() = k;
    Tensor values = at::empty(shape, logits.options()), columns = at::empty(shape, logits.options().dtype(at::kLong));
    shape.pop_back();
    Tensor lse = at::empty(shape, wide(logits)), scratch;
    if (const int64_t n = clg_top_logits_scratch_bytes(code_of(logits), r.rows, r.cols, k)) scratch = at::empty({n}, logits.options().dtype(at::kByte));
    check(clg_top_logits(code_of(logits), r.at, r.stride, r.rows, r.cols, k, temperature, values.data_ptr(), static_cast<int64_t *>(columns.data_ptr()),
                         lse.data_ptr(), scratch.defined() ? scratch.data_ptr() : nullptr, stream_of(logits)));
    return {values, columns, lse};
}

// ---- distillation ----------------------------------------------------------------------------------------------------------
struct DistillCall {
    Tensor values, columns, lse, mask;
    double temperature, weight;
    int64_t reduction;
    bool wanted;
    int call(bool backward, const Tensor &logits, const Tensor &upstream_or_loss, const Tensor &grad, const Tensor &applied, const Tensor &scratch) const
    {
        const Rows r(logits);
        const auto p = [](const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; };
        const auto run = [&](auto f, auto... between) {
            return f(code_of(logits), r.at, r.stride, values.data_ptr(), code_of(values), columns.data_ptr(), 8 * (int)columns.element_size(), p(lse),
                     lse.defined() ? code_of(lse) : CLG_F32, static_cast<const uint8_t *>(p(mask)), r.rows, r.cols, values.size(-1), temperature, weight,
                     (int)reduction, between..., p(grad), p(applied), p(scratch), stream_of(logits));
        };
        return backward ? run(clg_distill_backward, static_cast<const void *>(p(upstream_or_loss))) : run(clg_distill_forward, p(upstream_or_loss));
    }
};

// The forward call leaves the gradient for an upstream gradient of 1, from the same pass over the logits.  The first backward pass hands that
// tensor on -- the kernel looks at the upstream gradient and computes the rows again where it is another -- and later ones through a retained graph
// compute one of their own, since the first one's receiver may have changed it.  So does a backward pass of which only one side
// is recorded, or each into a graph of its own: one can be replayed without the other, and the tensor be written by nobody in between.
struct Distill : torch::autograd::Function<Distill> {
    static Tensor forward(AutogradContext *ctx, const Tensor &logits, const DistillCall *c)
    {
        const c10::OptionalDeviceGuard guard(logits.device());
        const Rows r(logits);
        const bool per_row = c->reduction == CLG_REDUCE_NONE;
        Tensor loss = at::empty(per_row ? logits.sizes().slice(0, logits.dim() - 1) : at::IntArrayRef(), wide(logits)), grad, applied, scratch;
        if (!per_row) scratch = at::empty({clg_distill_scratch_bytes(r.rows)}, logits.options().dtype(at::kByte));
        if (c->wanted && !per_row) {
            grad = at::empty(logits.sizes(), logits.options());
            applied = at::empty({r.rows}, wide(logits));
        }
        check(c->call(false, logits, loss, grad, applied, scratch));
        if (!c->wanted) return loss;
        ctx->save_for_backward({logits, c->values, c->columns, c->lse, c->mask});
        auto &kept = ctx->saved_data;
        kept["temperature"] = c->temperature;
        kept["weight"] = c->weight;
        kept["reduction"] = c->reduction;
        if (!per_row) {
            kept["grad"] = grad;
            kept["applied"] = applied;
            kept["scratch"] = scratch;                                // (one over the number of rows that the mask keeps)
            kept["recorded"] = recording();
        }
        return loss;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        static std::mutex taking;
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0];
        const c10::OptionalDeviceGuard guard(logits.device());
        Tensor grad, applied, scratch, up = grads[0].contiguous();
        DistillCall c{saved[1], saved[2], saved[3], saved[4]};
        {
            const std::lock_guard<std::mutex> lock(taking);
            auto &kept = ctx->saved_data;
            c.temperature = kept.at("temperature").toDouble(), c.weight = kept.at("weight").toDouble(), c.reduction = kept.at("reduction").toInt();
            const auto it = kept.find("grad");
            if (it != kept.end() && kept.at("recorded").toInt() == recording()) {
                grad = it->second.toTensor();
                applied = kept.at("applied").toTensor();
                scratch = kept.at("scratch").toTensor();
                for (const char *name : {"grad", "applied", "scratch"}) kept.erase(name);
            }
        }
        TORCH_CHECK(up.scalar_type() == wide(logits).dtype() && up.device() == logits.device(), "the loss's gradient must be ", wide(logits).dtype(), " on ",
                    logits.device());
        if (!grad.defined()) {
            grad = at::empty(logits.sizes(), logits.options());
            if (c.reduction == CLG_REDUCE_MEAN) scratch = at::empty({clg_distill_scratch_bytes(Rows(logits).rows)}, logits.options().dtype(at::kByte));
        }
        check(c.call(true, logits, up, grad, applied, scratch));
        return once({grad, Tensor()});
    }
};
Tensor distillation(const Tensor &logits, const Tensor &values, const Tensor &columns, const OptTensor &lse, const OptTensor &mask, double temperature,
                    double weight, int64_t reduction)
{
    const auto dense = [](const OptTensor &t) { return t ? t->detach().contiguous() : Tensor(); };
    const DistillCall c{dense(values), dense(columns), dense(lse), dense(mask), temperature, weight, reduction,
                        logits.requires_grad() && at::GradMode::is_enabled()};
    return Distill::apply(rows_of(logits), &c);
}

// ---- balance ---------------------------------------------------------------------------------------------------------------
struct BalanceCall {
    int64_t k;
    double weight;
    Tensor mask;
};
struct Segments {
    std::vector<const void *> at;
    std::vector<int64_t> rows, strides;
    explicit Segments(at::TensorList logits)
    {
        for (const Tensor &t : logits) {
            const Rows r(t);
            at.push_back(r.at), rows.push_back(r.rows), strides.push_back(r.stride);
        }
    }
};
struct Balance : torch::autograd::Function<Balance> {
    static variable_list forward(AutogradContext *ctx, at::TensorList logits, const BalanceCall *c)
    {
        const Tensor &first = logits[0];
        const c10::OptionalDeviceGuard guard(first.device());
        const int64_t n = (int64_t)logits.size(), experts = first.size(-1);
        const Segments s(logits);
        Tensor loss = at::empty({}, wide(first)), counts = at::empty({n, experts}, first.options().dtype(at::kLong)), coefs = at::empty({n, experts}, wide(first));
        Tensor scratch = at::empty({clg_balance_scratch_bytes(code_of(first), experts)}, first.options().dtype(at::kByte));
        check(clg_balance_forward(code_of(first), (int)n, s.at.data(), s.rows.data(), s.strides.data(), experts, c->k,
                                  c->mask.defined() ? static_cast<const uint8_t *>(c->mask.data_ptr()) : nullptr, c->weight, loss.data_ptr(),
                                  static_cast<int64_t *>(counts.data_ptr()), coefs.data_ptr(), scratch.data_ptr(), stream_of(first)));
        variable_list keep(logits.begin(), logits.end());
        keep.insert(keep.end(), {c->mask, coefs});
        ctx->save_for_backward(std::move(keep));
        ctx->mark_non_differentiable({counts});
        ctx->set_materialize_grads(false);
        return {loss, counts};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        const auto saved = ctx->get_saved_variables();
        const size_t n = saved.size() - 2;
        variable_list out(n + 1);
        if (!grads[0].defined()) return out;
        const Tensor &first = saved[0], &mask = saved[n], &coefs = saved[n + 1];
        const c10::OptionalDeviceGuard guard(first.device());
        const Tensor up = grads[0].contiguous();
        TORCH_CHECK(up.scalar_type() == coefs.scalar_type() && up.device() == first.device(), "the loss's gradient must be ", coefs.dtype(), " on ",
                    first.device());
        Segments s(at::TensorList(saved.data(), n));
        std::vector<void *> to(n);
        for (size_t i = 0; i < n; ++i) {
            if (ctx->needs_input_grad(i)) {
                out[i] = at::empty(saved[i].sizes(), saved[i].options());
                to[i] = out[i].data_ptr();
            } else {
                s.rows[i] = 0;
            }
        }
        check(clg_balance_backward(code_of(first), (int)n, s.at.data(), s.rows.data(), s.strides.data(), first.size(-1),
                                   mask.defined() ? static_cast<const uint8_t *>(mask.data_ptr()) : nullptr, coefs.data_ptr(), up.data_ptr(), to.data(),
                                   stream_of(first)));
        return once(std::move(out));
    }
};
std::tuple<Tensor, Tensor> balance(const std::vector<Tensor> &logits, int64_t k, const OptTensor &mask, double weight)
{
    variable_list dense;
    for (const Tensor &t : logits) dense.push_back(rows_of(t));
    const BalanceCall c{k, weight, mask ? mask->contiguous() : Tensor()};
    const auto out = Balance::apply(at::TensorList(dense), &c);
    return {out[0], out[1]};
}

// ---- cross entropy of group sums --------------------------------------------------------------------------------------------
struct GroupCeCall {
    Tensor targets;
    int64_t k;
    double tau, smoothing, weight;
    int64_t reduction;
    bool wanted;
};
// x [..., features] as the kernels read it: rows of dense features, or [features, rows] behind a transposed view
bool in_columns(const Tensor &x) { return x.dim() == 2 && !x.is_contiguous() && x.stride(0) == 1 && x.stride(1) == x.size(0); }
Tensor like_features(const Tensor &x)
{
    return in_columns(x) ? at::empty({x.size(1), x.size(0)}, x.options()).t() : at::empty(x.sizes(), x.options());
}
struct GroupCe : torch::autograd::Function<GroupCe> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const GroupCeCall *c)
    {
        const c10::OptionalDeviceGuard guard(x.device());
        const bool per_row = c->reduction == CLG_REDUCE_NONE, columns = in_columns(x);
        const Rows r(x);
        const auto room = [&](int64_t n) { return at::empty({n}, x.options().dtype(at::kByte)); };
        Tensor loss = at::empty(per_row ? x.sizes().slice(0, x.dim() - 1) : at::IntArrayRef(), wide(x)), grad;
        const Tensor kept = room(clg_group_ce_kept_bytes(code_of(x), columns, r.rows, r.cols, c->k)),
                     scratch = room(clg_group_ce_scratch_bytes(code_of(x), columns, r.rows, r.cols, c->k));
        if (c->wanted && !per_row) grad = like_features(x);
        check(clg_group_ce_forward(code_of(x), r.at, columns ? -1 : r.stride, r.rows, r.cols, c->k, c->targets.data_ptr(), 8 * (int)c->targets.element_size(),
                                   c->tau, c->smoothing, c->weight, (int)c->reduction, loss.data_ptr(), grad.defined() ? grad.data_ptr() : nullptr,
                                   kept.data_ptr(), scratch.data_ptr(), stream_of(x)));
        if (!c->wanted) return loss;
        ctx->save_for_backward({x, c->targets, kept});
        auto &data = ctx->saved_data;
        data["k"] = c->k;
        data["tau"] = c->tau;
        data["smoothing"] = c->smoothing;
        data["weight"] = c->weight;
        data["reduction"] = c->reduction;
        if (!per_row) {                                               // (handed on to the first backward pass, as Distill does)
            data["grad"] = grad;
            data["recorded"] = recording();
        }
        return loss;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        static std::mutex taking;
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &targets = saved[1], &kept = saved[2];
        const c10::OptionalDeviceGuard guard(x.device());
        const Tensor up = grads[0].contiguous();
        TORCH_CHECK(up.scalar_type() == wide(x).dtype() && up.device() == x.device(), "the loss's gradient must be ", wide(x).dtype(), " on ", x.device());
        Tensor grad;
        GroupCeCall c;
        {
            const std::lock_guard<std::mutex> lock(taking);
            auto &data = ctx->saved_data;
            c.k = data.at("k").toInt(), c.tau = data.at("tau").toDouble(), c.smoothing = data.at("smoothing").toDouble(), c.weight = data.at("weight").toDouble();
            c.reduction = data.at("reduction").toInt();
            const auto it = data.find("grad");
            if (it != data.end() && data.at("recorded").toInt() == recording()) {
                grad = it->second.toTensor();
                data.erase("grad");
            }
        }
        const bool has_grad = grad.defined();
        if (!has_grad) grad = like_features(x);
        const Rows r(x);
        check(clg_group_ce_backward(code_of(x), r.at, in_columns(x) ? -1 : r.stride, r.rows, r.cols, c.k, targets.data_ptr(), 8 * (int)targets.element_size(), c.tau,
                                    c.smoothing, c.weight, (int)c.reduction, up.data_ptr(), grad.data_ptr(), has_grad, kept.data_ptr(), stream_of(x)));
        return once({grad, Tensor()});
    }
};
Tensor group_ce(const Tensor &x, const Tensor &targets, int64_t k, double tau, double smoothing, double weight, int64_t reduction)
{
    const GroupCeCall c{targets.contiguous(), k, tau, smoothing, weight, reduction, x.requires_grad() && at::GradMode::is_enabled()};
    return GroupCe::apply(in_columns(x) ? x : rows_of(x), &c);
}

template <typename F>
void name_node(const char *name)
{
    static PyTypeObject type;
    torch::autograd::_initFunctionPyTypeObject(type, name, nullptr, nullptr);
    torch::autograd::registerCppFunction(typeid(torch::autograd::CppNode<F>), &type);
}

}  // namespace

void add_loss_nodes(pybind11::module_ &m)
{
    const auto no_gil = pybind11::call_guard<pybind11::gil_scoped_release>();
    name_node<Distill>("_DistillationBackward");
    name_node<Balance>("_BalanceBackward");
    name_node<GroupCe>("_GroupCrossEntropyBackward");
    m.def("group_ce", &group_ce, no_gil);
    m.def("top_logits", &top_logits, no_gil);
    m.def("distillation", &distillation, no_gil);
    m.def("balance", &balance, no_gil);
}
