// ops_torch.cpp -- the operators of libartemis_ops.so as functions on torch tensors: checks, memory, the current
// stream and autograd.  A call costs a few microseconds here; the same in Python took 60 to 130, longer
// than the kernels on all but large inputs, and a step over 320 tensors 0.7 ms.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <cmath>
#include <limits>

#include "artemis_ops.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<at::Tensor>;

int type_code(const at::Tensor &t, const char *what)
{
    switch (t.scalar_type()) {
    case at::kFloat: return ARTEMIS_OPS_F32;
    case at::kBFloat16: return ARTEMIS_OPS_BF16;
    case at::kHalf: return ARTEMIS_OPS_F16;
    default: TORCH_CHECK_TYPE(false, what, " must be float32, bfloat16 or float16, got ", t.scalar_type());
    }
}

// the framework's contract: contiguity is asserted
void assert_contiguous(const at::Tensor &t, const char *what)
{
    if (t.is_contiguous()) return;
    PyErr_Format(PyExc_AssertionError, "%s must be contiguous", what);
    throw pybind11::error_already_set();
}

void on_gpu(const at::Tensor &t)
{
    TORCH_CHECK_NOT_IMPLEMENTED(t.is_cuda(), "the operators run on HIP devices only, got a tensor on ", t.device());
}

void ok(int code, const char *what)
{
    TORCH_CHECK(code == 0, what, " failed (hipError ", code, "): ", artemis_ops_last_error());
}

void *stream_of(const at::Tensor &t)
{
    return (void *)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

const void *in(const at::Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *out(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
const float *in_f(const at::Tensor &t) { return (const float *)in(t); }
float *out_f(const at::Tensor &t) { return (float *)out(t); }

at::Tensor workspace_of(size_t bytes, const at::Tensor &like)
{
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}

// A parameter as the kernels read it: contiguous fp32 on the input's device.  Another floating type is widened through
// autograd, so that its gradient comes back in that type.
MaybeTensor parameter(const MaybeTensor &t, at::IntArrayRef shape, const at::Tensor &like, const char *what)
{
    if (!t || !t->defined()) return std::nullopt;
    type_code(*t, what);
    TORCH_CHECK_VALUE(t->sizes() == shape, what, " must be ", shape, ", got ", t->sizes());
    TORCH_CHECK_VALUE(t->device() == like.device(), what, " is on ", t->device(), ", the input on ", like.device());
    assert_contiguous(*t, what);
    return t->scalar_type() == at::kFloat ? t : t->to(at::kFloat);
}

// First derivatives only: where a graph of the backward pass is being built (create_graph), its results lead to an error.
variable_list once(variable_list grads)
{
    if (!at::GradMode::is_enabled()) return grads;
    variable_list given;
    for (auto &g : grads)
        if (g.defined()) given.push_back(g.detach().requires_grad_(true));
    auto node = std::make_shared<torch::autograd::DelayedError>(
        "artemis_amd's encoder operators have no second derivatives", (int64_t)given.size());
    variable_list kept = (*node)(std::move(given));
    size_t i = 0;
    for (auto &g : grads)
        if (g.defined()) g = kept[i++];
    return grads;
}

// The gradient node of the leaf that an edge leads to, itself or through copies: a parameter that was widened, an input that
// was realigned (below), or what a caller cast.
torch::autograd::AccumulateGrad *leaf_behind(const torch::autograd::Edge &edge)
{
    for (auto *node = edge.function.get(); node; node = node->next_edge(0).function.get()) {
        if (auto *leaf = dynamic_cast<torch::autograd::AccumulateGrad *>(node)) return leaf;
        const std::string name = node->name();
        if (node->num_outputs() != 1 || (name != "ToCopyBackward0" && name != "CloneBackward0")) return nullptr;
    }
    return nullptr;
}

// A leaf's gradient node is made with the first graph that has the leaf and lives with it.  Where that was on the default
// stream and is alive, a backward pass under capture makes torch wait for the capture on the default stream, which ends the
// capture, and may end the process: refused here, in front of that.
void no_outside_graph()
{
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    for (const auto &edge : node->next_edges()) {
        auto *leaf = leaf_behind(edge);
        if (!leaf) continue;
        const auto stream = leaf->stream();
        TORCH_CHECK(!stream || stream->id() != 0, "this backward pass is being captured while a graph of the same tensors that "
                    "was made on the default stream is alive: delete its outputs before the capture");
    }
}

// -------------------------------------------------------------------------------------------- layer norm

class LayerNorm : public torch::autograd::Function<LayerNorm> {
public:
    static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, const MaybeTensor &maybe_weight,
                              const MaybeTensor &maybe_bias, double eps, bool train)
    {
        const at::Tensor weight = maybe_weight.value_or(at::Tensor()), bias = maybe_bias.value_or(at::Tensor());
        const int64_t cols = x.size(-1), rows = cols ? x.numel() / cols : 0;
        const c10::DeviceGuard guard(x.device());
        at::Tensor y = at::empty_like(x), stats;
        if (train) stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
        float *mean = out_f(stats);
        ok(artemis_ops_layer_norm_forward(in(x), in_f(weight), in_f(bias), out(y), mean, mean ? mean + rows : nullptr, rows,
                                          cols, (float)eps, type_code(x, "x"), stream_of(x)),
           "artemis_ops_layer_norm_forward");
        if (train) {
            ctx->save_for_backward({x, weight, stats});
            ctx->saved_data["bias"] = bias.defined();
        }
        return y;
    }

    static variable_list backward(AutogradContext *ctx, variable_list dys)
    {
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &weight = saved[1], &stats = saved[2];
        if (!dys[0].defined()) return {{}, {}, {}, {}, {}};
        const int64_t cols = x.size(-1), rows = cols ? x.numel() / cols : 0;
        const int type = type_code(x, "x");
        const c10::DeviceGuard guard(x.device());
        no_outside_graph();
        const at::Tensor dy = dys[0].contiguous();
        const auto f32 = x.options().dtype(at::kFloat);
        at::Tensor dx, dw, db, workspace;
        if (ctx->needs_input_grad(0)) dx = at::empty_like(x);
        // (the tensors among the arguments are counted)
        if (weight.defined() && ctx->needs_input_grad(1)) dw = at::empty({cols}, f32);
        if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(1 + weight.defined())) db = at::empty({cols}, f32);
        size_t bytes = 0;
        if (dw.defined() || db.defined()) {
            bytes = artemis_ops_layer_norm_workspace_bytes(rows, cols, type);
            workspace = workspace_of(bytes, x);
        }
        const float *mean = in_f(stats);
        ok(artemis_ops_layer_norm_backward(in(x), in(dy), in_f(weight), mean, mean + rows, out(dx), out_f(dw), out_f(db),
                                           rows, cols, type, out(workspace), bytes, stream_of(x)),
           "artemis_ops_layer_norm_backward");
        return once({dx, dw, db, {}, {}});
    }
};

bool wants_grad(const at::Tensor &x, const MaybeTensor &a, const MaybeTensor &b)
{
    return at::GradMode::is_enabled() && (x.requires_grad() || (a && a->requires_grad()) || (b && b->requires_grad()));
}

at::Tensor layer_norm(const at::Tensor &x, const MaybeTensor &weight, const MaybeTensor &bias, double eps)
{
    type_code(x, "x");
    TORCH_CHECK_VALUE(x.dim() >= 1, "x must be (..., C)");
    TORCH_CHECK_VALUE(eps >= 0, "eps must be >= 0, got ", eps);
    const MaybeTensor w = parameter(weight, {x.size(-1)}, x, "weight"), b = parameter(bias, {x.size(-1)}, x, "bias");
    assert_contiguous(x, "x");
    on_gpu(x);
    return LayerNorm::apply(x, w, b, eps, wants_grad(x, w, b));
}

// --------------------------------------------------------------------------------------------- attention

// The kernels load four elements at once; a view that starts elsewhere is copied.
at::Tensor aligned(const at::Tensor &t)
{
    return (size_t)t.const_data_ptr() % (4 * t.element_size()) == 0 ? t : t.clone();
}

class WindowAttention : public torch::autograd::Function<WindowAttention> {
public:
    static at::Tensor forward(AutogradContext *ctx, const at::Tensor &qkv, const MaybeTensor &maybe_table,
                              const MaybeTensor &maybe_labels, const artemis_ops_window &w, bool train)
    {
        const at::Tensor table = maybe_table.value_or(at::Tensor()), labels = maybe_labels.value_or(at::Tensor());
        const c10::DeviceGuard guard(qkv.device());
        at::Tensor o = at::empty({w.B, w.D, w.H, w.W, (int64_t)w.heads * w.head_dim}, qkv.options()), lse;
        if (train)
            if (const size_t n = artemis_ops_window_attention_lse_count(&w))
                lse = at::empty({(int64_t)n}, qkv.options().dtype(at::kFloat));
        const size_t bytes = artemis_ops_window_attention_workspace_bytes(&w, 0, 0);
        const at::Tensor workspace = workspace_of(bytes, qkv);
        ok(artemis_ops_window_attention_forward(&w, in(qkv), in_f(table), (const int *)in(labels), out(o), out_f(lse),
                                                out(workspace), bytes, stream_of(qkv)),
           "artemis_ops_window_attention_forward");
        if (train) {
            // short windows: the backward pass computes the softmax again and reads neither output nor lse
            ctx->save_for_backward({qkv, table, labels, lse.defined() ? o : at::Tensor(), lse});
            ctx->saved_data["w"] = std::string((const char *)&w, sizeof(w));
        }
        return o;
    }

    static variable_list backward(AutogradContext *ctx, variable_list douts)
    {
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &qkv = saved[0], &table = saved[1], &labels = saved[2], &o = saved[3], &lse = saved[4];
        if (!douts[0].defined()) return {{}, {}, {}, {}, {}};
        artemis_ops_window w;
        const std::string packed = ctx->saved_data["w"].toStringRef();
        memcpy(&w, packed.data(), sizeof(w));
        const c10::DeviceGuard guard(qkv.device());
        no_outside_graph();
        const at::Tensor dout = aligned(douts[0].contiguous());
        const at::Tensor dqkv = at::empty_like(qkv);
        at::Tensor dtable;
        if (table.defined() && ctx->needs_input_grad(1)) dtable = at::empty_like(table);
        const size_t bytes = artemis_ops_window_attention_workspace_bytes(&w, 1, dtable.defined());
        const at::Tensor workspace = workspace_of(bytes, qkv);
        ok(artemis_ops_window_attention_backward(&w, in(qkv), in_f(table), (const int *)in(labels), in(o), in_f(lse), in(dout),
                                                 out(dqkv), out_f(dtable), out(workspace), bytes, stream_of(qkv)),
           "artemis_ops_window_attention_backward");
        return once({ctx->needs_input_grad(0) ? dqkv : at::Tensor(), dtable, {}, {}, {}});
    }
};

at::Tensor window_attention(const at::Tensor &qkv, const MaybeTensor &bias_table, const std::vector<int64_t> &window,
                            int64_t heads, const std::vector<int64_t> &shift, const MaybeTensor &labels, double outside,
                            std::optional<double> scale)
{
    const int type = type_code(qkv, "qkv");
    TORCH_CHECK_VALUE(qkv.dim() == 5, "qkv must be (B, D, H, W, 3 * C), got ", qkv.sizes());
    TORCH_CHECK_VALUE(window.size() == 3, "window must be (d, h, w), got ", window);
    TORCH_CHECK_VALUE(shift.size() == 3, "shift must be (d, h, w), got ", shift);
    const int64_t B = qkv.size(0), C3 = qkv.size(4);
    TORCH_CHECK_VALUE(heads >= 1 && heads <= 1024 && C3 % (3 * heads) == 0, "qkv's last dimension ", C3,
                      " is not 3 * num_heads * head_dim for ", heads, " heads (1 to 1024)");
    const int64_t hd = C3 / (3 * heads);
    TORCH_CHECK_VALUE(hd % 4 == 0 && hd >= 4 && hd <= 128, "head_dim ", hd, " must be a multiple of 4 up to 128");
    int64_t tokens = 1, entries = 1;
    for (int i = 0; i < 3; ++i) {
        TORCH_CHECK_VALUE(window[i] >= 1 && window[i] <= 4096, "window ", window, " must hold 1 to 4096 tokens");
        tokens *= window[i];
        entries *= 2 * window[i] - 1;
        TORCH_CHECK_VALUE(tokens <= 4096, "window ", window, " must hold 1 to 4096 tokens");
        TORCH_CHECK_VALUE(qkv.size(1 + i) % window[i] == 0, "map ", qkv.sizes().slice(1, 3), " is not a multiple of the window ",
                          window);
        TORCH_CHECK_VALUE(shift[i] >= 0 && shift[i] < window[i], "shift ", shift, " must lie in [0, window) for the window ",
                          window);
        TORCH_CHECK_VALUE(qkv.size(1 + i) <= std::numeric_limits<int>::max(), "the map is too large");
    }
    TORCH_CHECK_VALUE(B <= std::numeric_limits<int>::max(), "the batch is too large");
    TORCH_CHECK_VALUE(outside <= 0, "outside must be <= 0, got ", outside);
    const double s = scale ? *scale : 1.0 / std::sqrt((double)hd);
    TORCH_CHECK_VALUE(std::isfinite(s) && std::isfinite((float)s), "scale must be finite, got ", s);
    const MaybeTensor table = parameter(bias_table, {entries, heads}, qkv, "bias_table");
    int maps = 0;
    if (labels) {
        const at::Tensor &lab = *labels;
        TORCH_CHECK_TYPE(lab.scalar_type() == at::kInt, "labels must be int32, got ", lab.scalar_type());
        TORCH_CHECK_VALUE(lab.sizes() == qkv.sizes().slice(1, 3) || lab.sizes() == qkv.sizes().slice(0, 4), "labels must be ",
                          qkv.sizes().slice(1, 3), " or ", qkv.sizes().slice(0, 4), ", got ", lab.sizes());
        TORCH_CHECK_VALUE(lab.device() == qkv.device(), "labels are on ", lab.device(), ", qkv on ", qkv.device());
        assert_contiguous(lab, "labels");
        maps = lab.dim() == 4 && B > 1 ? (int)B : 1;
    }
    assert_contiguous(qkv, "qkv");
    on_gpu(qkv);
    const artemis_ops_window w{(int)B, (int)qkv.size(1), (int)qkv.size(2), (int)qkv.size(3), (int)heads, (int)hd,
                               (int)window[0], (int)window[1], (int)window[2], (int)shift[0], (int)shift[1], (int)shift[2],
                               maps, type, (float)s, (float)outside};
    const at::Tensor x = aligned(qkv);
    return WindowAttention::apply(x, table, labels, w, wants_grad(x, table, std::nullopt));
}

// ------------------------------------------------------------------------------------------------- AdamW

constexpr int64_t kGroup = 256;  // elements that share a base

// A Python list or tuple of tensors, read where it lies: a step over 318 tensors spends 92 us in copies of four
// such lists and their checks, 28 so.
class Tensors {
public:
    Tensors(const char *name, const pybind11::object &list) : name_(name)
    {
        held_ = pybind11::reinterpret_steal<pybind11::object>(PySequence_Fast(list.ptr(), "a list of tensors is wanted"));
        if (!held_) throw pybind11::error_already_set();
        items_ = PySequence_Fast_ITEMS(held_.ptr());
        size_ = (size_t)PySequence_Fast_GET_SIZE(held_.ptr());
        for (size_t i = 0; i < size_; ++i) TORCH_CHECK_TYPE(THPVariable_Check(items_[i]), name, "[", i, "] is not a tensor");
    }
    size_t size() const { return size_; }
    bool empty() const { return size_ == 0; }
    const char *name() const { return name_; }
    const at::Tensor &operator[](size_t i) const { return THPVariable_Unpack(items_[i]); }

private:
    const char *name_;
    pybind11::object held_;
    PyObject **items_;
    size_t size_;
};

void check_list(const Tensors &ts, const Tensors &params, at::ScalarType type, bool groups)
{
    TORCH_CHECK_VALUE(ts.size() == params.size(), params.size(), " ", params.name(), " but ", ts.size(), " ", ts.name());
    const at::Device device = params[0].device();
    for (size_t i = 0; i < ts.size(); ++i) {
        const at::Tensor &t = ts[i];
        TORCH_CHECK_TYPE(t.scalar_type() == type, ts.name(), "[", i, "] must be ", type, ", got ", t.scalar_type());
        const int64_t count = params[i].numel(), want = groups ? (count + kGroup - 1) / kGroup : count;
        TORCH_CHECK_VALUE(t.numel() == want, ts.name(), "[", i, "] has ", t.numel(), " elements, ", want, " are wanted");
        TORCH_CHECK_VALUE(t.device() == device, ts.name(), "[", i, "] is on ", t.device(), ", ", params.name(), "[0] on ", device);
        assert_contiguous(t, ts.name());
    }
}

// What is written, in one list or in two: two workgroups would update it at once
class Distinct {
public:
    explicit Distinct(size_t most)
    {
        size_t n = 16;
        while (n < 2 * most) n *= 2;
        seen_.resize(n);
    }
    void add(const Tensors &ts)
    {
        const size_t mask = seen_.size() - 1;
        for (size_t i = 0; i < ts.size(); ++i) {
            if (ts[i].numel() == 0) continue;
            const void *p = ts[i].const_data_ptr();
            size_t at = ((size_t)p * 0x9E3779B97F4A7C15ull >> 32) & mask;
            for (; seen_[at]; at = (at + 1) & mask)
                TORCH_CHECK_VALUE(seen_[at] != p, ts.name(), " holds a tensor that was given twice");
            seen_[at] = p;
        }
    }

private:
    std::vector<const void *> seen_;  // at most half full
};

void adamw(const pybind11::object &param_list, const pybind11::object &grad_list, const pybind11::object &m_list,
           const pybind11::object &v_list, const pybind11::object &m_base_list, const pybind11::object &v_base_list, int bits,
           int64_t step, double lr, double beta1, double beta2, double eps, double weight_decay, int64_t seed)
{
    const Tensors params("params", param_list), grads("grads", grad_list), m("exp_avgs", m_list), v("exp_avg_sqs", v_list);
    const Tensors m_base("exp_avg_bases", m_base_list), v_base("exp_avg_sq_bases", v_base_list);
    if (params.empty() && grads.empty()) return;
    TORCH_CHECK_VALUE(!params.empty(), "no params but ", grads.size(), " grads");
    const int type = type_code(params[0], "params");
    const at::ScalarType kind = bits == 32 ? at::kFloat : at::kByte;
    check_list(params, params, params[0].scalar_type(), false);
    check_list(grads, params, params[0].scalar_type(), false);
    check_list(m, params, kind, false);
    check_list(v, params, kind, false);
    if (bits == 8) {
        check_list(m_base, params, at::kInt, true);
        check_list(v_base, params, at::kInt, true);
    }
    Distinct distinct(5 * params.size());
    distinct.add(params);
    distinct.add(m);
    distinct.add(v);
    if (bits == 8) {
        distinct.add(m_base);
        distinct.add(v_base);
    }
    TORCH_CHECK_VALUE(step >= 1, "step must be a whole number >= 1, got ", step);
    on_gpu(params[0]);
    std::vector<artemis_ops_tensor> list(params.size());
    for (size_t i = 0; i < params.size(); ++i)
        list[i] = {params[i].data_ptr(), grads[i].const_data_ptr(), m[i].data_ptr(), v[i].data_ptr(),
                   bits == 8 ? (int *)m_base[i].data_ptr() : nullptr, bits == 8 ? (int *)v_base[i].data_ptr() : nullptr,
                   params[i].numel()};
    const c10::DeviceGuard guard(params[0].device());
    ok(artemis_ops_adamw(list.data(), (int)list.size(), type, bits, lr, beta1, beta2, eps, weight_decay, step, (unsigned)seed,
                         stream_of(params[0])),
       "artemis_ops_adamw");
    // what autograd saved of them is out of date
    for (size_t i = 0; i < params.size(); ++i)
        if (!params[i].is_inference()) params[i].unsafeGetTensorImpl()->bump_version();
}

std::vector<at::Tensor> moments_from_8bit(const pybind11::object &code_list, const pybind11::object &base_list, bool is_signed)
{
    const Tensors codes("codes", code_list), bases("bases", base_list);
    if (codes.empty() && bases.empty()) return {};
    TORCH_CHECK_VALUE(!codes.empty(), "no codes but ", bases.size(), " bases");
    check_list(codes, codes, at::kByte, false);
    check_list(bases, codes, at::kInt, true);
    on_gpu(codes[0]);
    const c10::DeviceGuard guard(codes[0].device());
    std::vector<at::Tensor> values;
    std::vector<artemis_ops_tensor> list;
    for (size_t i = 0; i < codes.size(); ++i) {
        values.push_back(at::empty(codes[i].sizes(), codes[i].options().dtype(at::kFloat)));
        list.push_back({values[i].data_ptr(), nullptr, codes[i].data_ptr(), nullptr, (int *)bases[i].data_ptr(), nullptr,
                        codes[i].numel()});
    }
    ok(artemis_ops_moments_from_8bit(list.data(), (int)list.size(), is_signed, stream_of(codes[0])),
       "artemis_ops_moments_from_8bit");
    return values;
}

}  // namespace

PYBIND11_MODULE(_artemis_ops, m)
{
    m.def("layer_norm", &layer_norm);
    m.def("window_attention", &window_attention);
    m.def("adamw", &adamw);
    m.def("moments_from_8bit", &moments_from_8bit);
    // whether the tensor is a leaf that wants a gradient, or a copy of one, as a captured backward pass looks for it
    m.def("has_leaf", [](const at::Tensor &t) { return leaf_behind(torch::autograd::impl::gradient_edge(t)) != nullptr; });
}
