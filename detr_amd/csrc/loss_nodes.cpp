// Host side of the losses that have a node of their own in the autograd graph (detr_amd.losses: the classification losses that
// keep 8 bits per logit, the balance loss of expert routers): checks of arguments, workspaces, the call of the library's entry
// point, and the node whose backward pass is another such call.
//
// As Python functions the same nodes cost more than their kernels at the criterion's ordinary sizes: the backward pass runs in
// the autograd engine's thread, which has to take the interpreter lock from the caller's and hand it back.  Host time of
// forward and backward of a focal loss of 4 x 300 x 91 logits: 117 us as Python nodes, 55 us as these (of which the engine
// itself takes some 40); of the balance loss of 1 x 300 x 8: 141 us and 63 us.  Nothing here holds the lock in the backward
// pass (but for hooks of Python on saved tensors).
//
// No GPU code: the kernels are reached through the addresses of libdetr_match.so's entry points, handed over once by `bind`.
// Built against one torch version, which the module names (`built_for_torch`); the Python code refuses it under any other.
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include "detr_match.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptionalTensors = std::vector<std::optional<Tensor>>;

struct Entries {
    decltype(&dm_focal_loss_saved) focal_saved;
    decltype(&dm_focal_loss_from_saved) focal_from_saved;
    decltype(&dm_cross_entropy_saved) ce_saved;
    decltype(&dm_cross_entropy_from_saved) ce_from_saved;
    decltype(&dm_balance_workspace) balance_workspace;
    decltype(&dm_balance_loss) balance_loss;
    decltype(&dm_balance_backward) balance_backward;
    decltype(&dm_expert_counts) expert_counts;
    decltype(&dm_strerror) strerror;
    decltype(&dm_last_hip_error) last_hip_error;
} g;

void bind(const std::unordered_map<std::string, uintptr_t> &addresses)
{
    auto take = [&](const char *name, auto &entry) {
        const auto it = addresses.find(name);
        TORCH_CHECK(it != addresses.end() && it->second, "no entry point ", name);
        entry = reinterpret_cast<std::decay_t<decltype(entry)>>(it->second);
    };
    take("dm_focal_loss_saved", g.focal_saved);
    take("dm_focal_loss_from_saved", g.focal_from_saved);
    take("dm_cross_entropy_saved", g.ce_saved);
    take("dm_cross_entropy_from_saved", g.ce_from_saved);
    take("dm_balance_workspace", g.balance_workspace);
    take("dm_balance_loss", g.balance_loss);
    take("dm_balance_backward", g.balance_backward);
    take("dm_expert_counts", g.expert_counts);
    take("dm_strerror", g.strerror);
    take("dm_last_hip_error", g.last_hip_error);
}

// The exceptions of detr_amd._lib.check.
void check(int rc, const char *what)
{
    if (rc == DM_OK) return;
    TORCH_CHECK_NOT_IMPLEMENTED(rc != DM_E_UNSUPPORTED, what, ": ", g.strerror(rc), " (see include/detr_match.h)");
    TORCH_CHECK(rc != DM_E_LAUNCH, what, ": ", g.strerror(rc), ": ", g.last_hip_error());
    TORCH_CHECK(false, what, ": ", g.strerror(rc));
}

void *current_stream(const at::Device &device) { return c10::hip::getCurrentHIPStream(device.index()).stream(); }

int dtype_code(const Tensor &t, const char *what)
{
    switch (t.scalar_type()) {
    case at::kFloat: return DM_F32;
    case at::kBFloat16: return DM_BF16;
    case at::kHalf: return DM_F16;
    default: TORCH_CHECK_TYPE(false, what, " must be float32, bfloat16 or float16, got ", t.scalar_type());
    }
    return -1;
}

// What works below autograd does not show: a tangent would be dropped without a word, and a trace would hold the allocations
// without the kernels between them.
void refuse_tracing()
{
    const bool proxies = c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value();
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() && !proxies,
                                "detr_amd.losses: this call cannot be traced (torch.jit.trace, torch.fx of tensors)");
}
void refuse_tangent(const Tensor &t)
{
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(),
                                "detr_amd.losses: this loss has no derivative for forward-mode differentiation");
}

// A node that is used once unless the graph is retained, and whose gradients have no gradients of their own.
struct LossNode : torch::autograd::Node {
    variable_list apply(variable_list &&grads) override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE);
        // (the hooks of saved tensors may run anything, a whole forward pass among it: not below autograd)
        const variable_list saved = unpack(grads);
        variable_list out;
        {
            const at::AutoDispatchBelowADInplaceOrView below;
            out = backward(grads, saved);
        }
        if (!at::GradMode::is_enabled()) return out;
        // create_graph=True: what would differentiate these gradients again is refused when it is tried
        for (auto &t : out)
            if (t.defined()) t = t.detach().set_requires_grad(true);
        return torch::autograd::DelayedError(
            "detr_amd.losses: the gradient of this loss is not differentiable (a double backward was asked for)",
            static_cast<int64_t>(out.size())).apply(std::move(out));
    }
    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        released = true;
        drop();
    }
    // What the backward pass needs of the saved tensors, in an order of the node's own.
    virtual variable_list unpack(const variable_list &grads) = 0;
    virtual variable_list backward(const variable_list &grads, const variable_list &saved) = 0;
    virtual void drop() = 0;
    bool released = false;
};

// A saved tensor, and what the kernels take it for: a hook (torch.autograd.graph.saved_tensors_hooks) may hand back another.
struct Saved {
    SavedVariable variable;
    at::Device device = at::kCPU;
    at::ScalarType type = at::kByte;
    at::DimVector sizes;

    Saved() = default;
    // (a tensor of inference mode cannot be saved as it is)
    explicit Saved(const Tensor &t) : variable(t.is_inference() ? t.clone() : t, false), device(t.device()), type(t.scalar_type()), sizes(t.sizes()) {}
    Tensor unpack() const
    {
        const Tensor t = variable.unpack();
        TORCH_CHECK(t.defined() && t.device() == device && t.scalar_type() == type && t.sizes() == at::IntArrayRef(sizes),
                    "detr_amd.losses: a hook has handed back another saved tensor than ", type, " ", at::IntArrayRef(sizes), " on ", device);
        return t;
    }
};

bool wants_grad(const std::vector<Tensor> &inputs)
{
    if (!at::GradMode::is_enabled()) return false;
    for (const auto &t : inputs)
        if (t.requires_grad()) return true;
    return false;
}

// ---- the classification losses that keep 8 bits per logit ----

struct ClsCall {
    bool ce;
    double alpha, gamma;
    std::vector<double> scales;      // focal: one per set
    int64_t ignore_index;
    bool use_ignore;
};

struct ClsNode : LossNode {
    ClsCall call;
    struct Set {
        at::TensorOptions options;
        at::DimVector shape;
        int dtype;
        int64_t rows, C, n, data;      // bytes of `codes` before the heads or steps
        Saved codes, cls;              // (of the sets that need a gradient)
    };
    std::vector<Set> sets;
    Saved weight;
    bool weighted = false;
    Saved out;                         // cross entropy: [S, 2], 1 / sum of the weights in the second column

    std::string name() const override { return call.ce ? "CrossEntropy8Backward" : "FocalLoss8Backward"; }
    void drop() override
    {
        for (auto &s : sets) {
            s.codes.variable.reset_data();
            s.cls.variable.reset_data();
        }
        weight.variable.reset_data();
        out.variable.reset_data();
    }
    variable_list unpack(const variable_list &grads) override
    {
        variable_list saved(2 * sets.size() + 2);
        if (!grads[0].defined()) return saved;
        bool any = false;
        for (size_t i = 0; i < sets.size(); ++i) {
            if (!task_should_compute_output(i) || sets[i].n == 0) continue;
            saved[2 * i] = sets[i].codes.unpack();
            saved[2 * i + 1] = sets[i].cls.unpack();
            any = true;
        }
        if (any && weighted) saved[2 * sets.size()] = weight.unpack();
        if (any && call.ce) saved[2 * sets.size() + 1] = out.unpack();
        return saved;
    }
    variable_list backward(const variable_list &grads, const variable_list &saved) override
    {
        variable_list result(sets.size());
        if (!grads[0].defined()) return result;
        const Tensor upstream = grads[0].contiguous();
        const c10::DeviceGuard guard(upstream.device());
        void *stream = current_stream(upstream.device());
        auto dense = [](const Tensor &t) { return t.defined() ? t.contiguous() : t; };
        const Tensor w = dense(saved[2 * sets.size()]), sums = dense(saved[2 * sets.size() + 1]);
        for (size_t i = 0; i < sets.size(); ++i) {
            if (!task_should_compute_output(i)) continue;
            Set &s = sets[i];
            Tensor grad = at::empty(s.shape, s.options);
            result[i] = grad;
            if (s.n == 0) continue;
            const Tensor bytes = dense(saved[2 * i]), cls = dense(saved[2 * i + 1]);
            const auto *codes = bytes.const_data_ptr<uint8_t>();
            const auto *g_loss = static_cast<const float *>(upstream.const_data_ptr()) + i;
            if (call.ce)
                check(g.ce_from_saved(codes, reinterpret_cast<const int8_t *>(codes + s.data), s.dtype, cls.const_data_ptr<int64_t>(),
                                      w.defined() ? w.const_data_ptr<float>() : nullptr, s.rows, static_cast<int>(s.C), call.ignore_index,
                                      sums.const_data_ptr<float>() + 2 * i + 1, g_loss, grad.mutable_data_ptr(), stream),
                      "dm_cross_entropy_from_saved");
            else
                check(g.focal_from_saved(codes, reinterpret_cast<const int32_t *>(codes + s.data), s.dtype, cls.const_data_ptr<int64_t>(),
                                         s.rows, static_cast<int>(s.C), static_cast<float>(call.alpha), static_cast<float>(call.gamma),
                                         static_cast<float>(call.scales[i]), call.ignore_index, call.use_ignore, g_loss,
                                         grad.mutable_data_ptr(), stream),
                      "dm_focal_loss_from_saved");
        }
        return result;
    }
};

// [S] losses of S sets; of a single one as a 0-dim tensor if asked for.
Tensor cls_losses(const std::vector<Tensor> &logits, const std::vector<Tensor> &maps, const std::optional<Tensor> &weight_in,
                  const ClsCall &call, bool scalar, const Tensor &status)
{
    const size_t S = logits.size();
    TORCH_CHECK_VALUE(S > 0 && maps.size() == S, "one class map for every set of logits");
    refuse_tracing();
    for (const auto &x : logits) refuse_tangent(x);
    if (weight_in) refuse_tangent(*weight_in);
    const at::Device device = logits[0].device();
    for (size_t i = 0; i < S; ++i) {
        const Tensor &x = logits[i], &cls = maps[i];
        TORCH_CHECK(x.is_cuda(), "detr_amd.losses: the classification loss runs on the GPU (there is no CPU path)");
        dtype_code(x, "logits");
        TORCH_CHECK_TYPE(cls.scalar_type() == at::kLong && cls.device() == x.device() && x.device() == device,
                         "target_cls must be an int64 tensor on the device of the logits");
        TORCH_CHECK_VALUE(x.dim() >= 1 && x.sizes().slice(0, x.dim() - 1) == cls.sizes(), "logits ", x.sizes(), " must be target_cls ",
                          cls.sizes(), " + [C]");
        TORCH_CHECK_VALUE(x.size(-1) >= 1, "logits of no class");
        TORCH_CHECK_NOT_IMPLEMENTED(x.size(-1) < (1ll << 31) && x.numel() < (1ll << 31), "rows * C must be below 2^31");
    }
    const bool grad = wants_grad(logits);
    std::shared_ptr<ClsNode> node;
    if (grad) {
        node = std::shared_ptr<ClsNode>(new ClsNode(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(logits));
        node->call = call;
        node->sets.resize(S);
    }
    std::optional<at::AutoDispatchBelowADInplaceOrView> below(std::in_place);
    const c10::DeviceGuard guard(device);
    Tensor weight;
    if (weight_in) {
        TORCH_CHECK_VALUE(weight_in->scalar_type() == at::kFloat && weight_in->device() == device && weight_in->dim() == 1,
                          "weight must be a float32 [C] tensor on the device of the logits");
        for (const auto &x : logits)
            TORCH_CHECK_VALUE(weight_in->size(0) == x.size(-1), "weight must be a float32 [C] tensor on the device of the logits");
        weight = weight_in->contiguous();
    }
    const auto bytes = at::TensorOptions().dtype(at::kByte).device(device);
    const auto floats = bytes.dtype(at::kFloat);
    // (the sets of a call run one after the other on the stream: one workspace)
    const Tensor partials = at::empty({DM_CLS_LOSS_PARTIALS}, bytes.dtype(at::kDouble));
    Tensor out = at::empty({static_cast<int64_t>(S), 2}, floats);
    void *stream = current_stream(device);
    std::vector<Tensor> kept(2 * S);                   // codes and classes
    for (size_t i = 0; i < S; ++i) {
        const Tensor x = logits[i].contiguous(), cls = maps[i].contiguous();
        const int dtype = dtype_code(x, "logits");
        const int64_t n = x.numel(), rows = cls.numel(), C = x.size(-1);
        const int64_t blocks = (n + 127) / 128, data = call.ce ? n : 128 * blocks, marks = call.ce ? rows : 4 * blocks;
        Tensor codes;
        uint8_t *codes_ptr = nullptr, *marks_ptr = nullptr;
        if (grad && logits[i].requires_grad()) {
            codes = at::empty({data + marks}, bytes);
            if (n) {
                codes_ptr = codes.mutable_data_ptr<uint8_t>();
                marks_ptr = codes_ptr + data;
            }
        }
        float *loss_out = out.mutable_data_ptr<float>() + 2 * i;
        if (call.ce)
            check(g.ce_saved(x.const_data_ptr(), dtype, cls.const_data_ptr<int64_t>(), weight.defined() ? weight.const_data_ptr<float>() : nullptr,
                             rows, static_cast<int>(C), call.ignore_index, loss_out, codes_ptr, reinterpret_cast<int8_t *>(marks_ptr),
                             partials.mutable_data_ptr<double>(), status.mutable_data_ptr<int32_t>(), stream),
                  "dm_cross_entropy_saved");
        else
            check(g.focal_saved(x.const_data_ptr(), dtype, cls.const_data_ptr<int64_t>(), rows, static_cast<int>(C),
                                static_cast<float>(call.alpha), static_cast<float>(call.gamma), static_cast<float>(call.scales[i]),
                                call.ignore_index, call.use_ignore, loss_out, codes_ptr, reinterpret_cast<int32_t *>(marks_ptr),
                                partials.mutable_data_ptr<double>(), status.mutable_data_ptr<int32_t>(), stream),
                  "dm_focal_loss_saved");
        if (grad) {
            ClsNode::Set &s = node->sets[i];
            s.options = x.options();
            s.shape = at::DimVector(logits[i].sizes());
            s.dtype = dtype;
            s.rows = rows;
            s.C = C;
            s.n = n;
            s.data = data;
            if (codes.defined()) {
                kept[2 * i] = codes;
                kept[2 * i + 1] = cls;
            }
        }
    }
    Tensor losses = scalar ? out.select(1, 0).select(0, 0) : out.select(1, 0);
    if (grad) {
        below.reset();                                 // (saving may run hooks)
        for (size_t i = 0; i < S; ++i) {
            if (!kept[2 * i].defined()) continue;
            node->sets[i].codes = Saved(kept[2 * i]);
            node->sets[i].cls = Saved(kept[2 * i + 1]);
        }
        if (weight.defined()) {
            node->weight = Saved(weight);
            node->weighted = true;
        }
        // (a version of its own: the losses, which may be changed in place, are the other column)
        if (call.ce) node->out = Saved(out.variable_data());
        torch::autograd::set_history(losses, node);
    }
    return losses;
}

Tensor focal_losses(const std::vector<Tensor> &logits, const std::vector<Tensor> &maps, double alpha, double gamma,
                    const std::vector<double> &scales, std::optional<int64_t> ignore_index, bool scalar, const Tensor &status)
{
    TORCH_CHECK_VALUE(scales.size() == logits.size(), "one scale for every set of logits");
    TORCH_CHECK_VALUE(!(gamma < 0.0), "gamma must not be below zero with saved_bits=8, got ", gamma);
    return cls_losses(logits, maps, std::nullopt, ClsCall{false, alpha, gamma, scales, ignore_index.value_or(0), ignore_index.has_value()},
                      scalar, status);
}

Tensor cross_entropies(const std::vector<Tensor> &logits, const std::vector<Tensor> &maps, const std::optional<Tensor> &weight,
                       int64_t ignore_index, bool scalar, const Tensor &status)
{
    return cls_losses(logits, maps, weight, ClsCall{true, 0.0, 0.0, {}, ignore_index, false}, scalar, status);
}

// ---- the status word of a call inside a capture ----

// An int32 zero that is no part of the graph that the current stream captures: neither its memory nor its clearing.  From a
// stream that captures nothing (of the pool that the capturing one may itself be of), while this thread may allocate and wait.
Tensor zero_word_outside_capture(int64_t device_index)
{
    const auto index = static_cast<c10::DeviceIndex>(device_index);
    const c10::hip::HIPGuard device(index);
    c10::hip::HIPStreamCaptureModeGuard relaxed(hipStreamCaptureModeRelaxed);
    for (int tries = 0; tries < 64; ++tries) {
        const c10::hip::HIPStream stream = c10::hip::getStreamFromPool(/*isHighPriority=*/false, index);
        const c10::hip::HIPStreamGuard on(stream);
        if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None) continue;
        const Tensor word = at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, index));
        stream.synchronize();
        return word;
    }
    TORCH_CHECK(false, "detr_amd.losses: no stream outside the capture");
}

// ---- the balance loss of expert routers ----

struct RouterCall {
    int dtype;
    int64_t S, B, E, top_k;
    int sigmoid, per_image;
    int64_t groups() const { return per_image ? S * B : S; }
    at::DimVector shape(bool experts) const
    {
        at::DimVector d{S};
        if (per_image) d.push_back(B);
        if (experts) d.push_back(E);
        return d;
    }
};

// Elements from one image to the next of a [B, Q, E] tensor whose rows are dense inside every image: 0 when it is contiguous,
// -1 when the kernels cannot read it in place.
int64_t image_stride(const Tensor &t)
{
    if (t.is_contiguous()) return 0;
    if (t.stride(2) != 1 || t.stride(1) != t.size(2)) return -1;
    if (t.size(0) <= 1) return 0;
    return t.stride(0) >= t.size(1) * t.size(2) ? t.stride(0) : -1;
}

// The logits as the kernels read them (in place where the rows of an image are dense), their masks and indices.
struct Routers {
    std::vector<Tensor> logits, masks, experts;

    Routers(const std::vector<Tensor> &in, const OptionalTensors &mask, const OptionalTensors &given, RouterCall &call)
    {
        TORCH_CHECK_VALUE(!in.empty(), "no router logits");
        const Tensor &first = in[0];
        TORCH_CHECK(first.is_cuda(), "detr_amd.losses: the balance loss runs on the GPU (there is no CPU path)");
        call.dtype = dtype_code(first, "router logits");
        TORCH_CHECK_VALUE(first.dim() == 3, "router logits must be [B, Q, E], got ", first.sizes());
        call.S = static_cast<int64_t>(in.size());
        call.B = first.size(0);
        call.E = first.size(2);
        TORCH_CHECK_VALUE(call.E >= 1, "router logits for no expert");
        const bool with_experts = given[0].has_value();
        TORCH_CHECK_VALUE(call.top_k >= 1 && (with_experts || call.top_k <= call.E),
                          "top_k must be a whole number from 1 to the number of experts (", call.E, "), got ", call.top_k);
        TORCH_CHECK_NOT_IMPLEMENTED(call.S < (1ll << 31) && call.B < (1ll << 31) && call.E < (1ll << 31) && call.top_k < (1ll << 31),
                                    "sets, images, experts and top_k must be below 2^31");
        logits.reserve(in.size());
        masks.resize(in.size());
        experts.resize(in.size());
        for (size_t i = 0; i < in.size(); ++i) {
            const Tensor &x = in[i];
            TORCH_CHECK_TYPE(x.scalar_type() == first.scalar_type() && x.device() == first.device(),
                             "the router logits of a call must share their type and device");
            TORCH_CHECK_VALUE(x.dim() == 3 && x.size(0) == call.B && x.size(2) == call.E,
                              "the router logits of a call must be [B, Q, E] with the same B and E");
            TORCH_CHECK_NOT_IMPLEMENTED(x.size(1) < (1ll << 31), "Q must be below 2^31");
            logits.push_back(image_stride(x) >= 0 ? x : x.contiguous());
            if (mask[i]) {
                TORCH_CHECK_TYPE(mask[i]->scalar_type() == at::kBool && mask[i]->device() == x.device(),
                                 "mask must be a bool tensor on the device of the router logits");
                TORCH_CHECK_VALUE(mask[i]->sizes() == x.sizes().slice(0, 2), "mask must be [B, Q] = ", x.sizes().slice(0, 2), ", got ",
                                  mask[i]->sizes());
                masks[i] = mask[i]->contiguous();
            }
            TORCH_CHECK_VALUE(given[i].has_value() == with_experts, "experts for all sets of the call or for none");
            if (with_experts) {
                TORCH_CHECK_TYPE(given[i]->scalar_type() == at::kLong && given[i]->device() == x.device(),
                                 "experts must be an int64 tensor on the device of the router logits");
                TORCH_CHECK_VALUE(given[i]->dim() == 3 && given[i]->size(0) == call.B && given[i]->size(1) == x.size(1) &&
                                      given[i]->size(2) == call.top_k,
                                  "experts must be [B, Q, top_k] = [", call.B, ", ", x.size(1), ", ", call.top_k, "], got ", given[i]->sizes());
                experts[i] = given[i]->contiguous();
            }
        }
    }
};

void describe(std::vector<DmRouterSet> &sets, size_t i, const Tensor &x, const Tensor &mask, const Tensor &experts, Tensor *grad)
{
    sets[i] = DmRouterSet{x.const_data_ptr(), mask.defined() ? static_cast<const uint8_t *>(mask.const_data_ptr()) : nullptr,
                          experts.defined() ? experts.const_data_ptr<int64_t>() : nullptr, grad ? grad->mutable_data_ptr() : nullptr,
                          image_stride(x), static_cast<int32_t>(x.size(1)), 0};
}

Tensor workspace_for(const std::vector<DmRouterSet> &sets, const RouterCall &c, const at::TensorOptions &bytes)
{
    const int64_t need = g.balance_workspace(sets.data(), static_cast<int>(c.S), static_cast<int>(c.B), static_cast<int>(c.E), c.per_image);
    if (need < 0) check(static_cast<int>(need), "dm_balance_workspace");
    return at::empty({need}, bytes);
}

struct BalanceNode : LossNode {
    RouterCall call;
    std::vector<Saved> logits, masks;      // (of the sets that need a gradient)
    std::vector<char> masked;
    Saved kept;       // slope [groups, E], then 1 / n [groups]

    std::string name() const override { return "BalanceLossesBackward"; }
    void drop() override
    {
        for (auto &v : logits) v.variable.reset_data();
        for (auto &v : masks) v.variable.reset_data();
        kept.variable.reset_data();
    }
    static bool any(const variable_list &grads) { return grads[0].defined() || (grads.size() > 1 && grads[1].defined()); }
    variable_list unpack(const variable_list &grads) override
    {
        const size_t S = logits.size();
        variable_list saved(2 * S + 1);
        if (!any(grads)) return saved;
        for (size_t i = 0; i < S; ++i) {
            if (!task_should_compute_output(i)) continue;
            saved[2 * i] = logits[i].unpack();
            if (masked[i]) saved[2 * i + 1] = masks[i].unpack();
        }
        saved[2 * S] = kept.unpack();
        return saved;
    }
    variable_list backward(const variable_list &grads, const variable_list &saved) override
    {
        const size_t S = logits.size();
        variable_list result(S);
        if (!any(grads)) return result;
        const Tensor gb = grads[0].defined() ? grads[0].contiguous() : Tensor();
        const Tensor gz = grads.size() > 1 && grads[1].defined() ? grads[1].contiguous() : Tensor();
        const Tensor shares = saved[2 * S].contiguous();
        const c10::DeviceGuard guard(shares.device());
        std::vector<DmRouterSet> sets(S);
        std::vector<Tensor> held(2 * S);
        for (size_t i = 0; i < S; ++i) {
            const Tensor &x = saved[2 * i];
            if (!x.defined()) continue;
            held[2 * i] = image_stride(x) >= 0 ? x : x.contiguous();
            if (masked[i]) held[2 * i + 1] = saved[2 * i + 1].contiguous();
            result[i] = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
            describe(sets, i, held[2 * i], held[2 * i + 1], Tensor(), &result[i]);
        }
        const float *slope = shares.const_data_ptr<float>();
        const float *inv_rows = slope + call.groups() * call.E;
        const size_t groups = call.per_image ? call.B : 1;      // of a set
        // (a call for each run of sets that need a gradient: one, unless some in between need none)
        for (size_t i = 0, end; i < S; i = end) {
            end = i + 1;
            if (!result[i].defined()) continue;
            while (end < S && result[end].defined()) ++end;
            check(g.balance_backward(sets.data() + i, static_cast<int>(end - i), static_cast<int>(call.B), static_cast<int>(call.E),
                                     call.dtype, call.sigmoid, call.per_image, slope + i * groups * call.E, inv_rows + i * groups,
                                     gb.defined() ? gb.const_data_ptr<float>() + i * groups : nullptr,
                                     gz.defined() ? gz.const_data_ptr<float>() + i * groups : nullptr, current_stream(shares.device())),
                  "dm_balance_backward");
        }
        return result;
    }
};

std::tuple<Tensor, std::optional<Tensor>, Tensor> balance_losses(const std::vector<Tensor> &in, int64_t top_k, const OptionalTensors &mask,
                                                                 const OptionalTensors &given, const std::optional<Tensor> &counts_in,
                                                                 bool sigmoid, bool per_image, const Tensor &status)
{
    RouterCall c{};
    c.top_k = top_k;
    c.sigmoid = sigmoid;
    c.per_image = per_image;
    refuse_tracing();
    for (const auto &x : in) refuse_tangent(x);
    const bool grad = wants_grad(in);
    std::shared_ptr<BalanceNode> node;
    if (grad) {
        node = std::shared_ptr<BalanceNode>(new BalanceNode(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(in));
    }
    std::optional<at::AutoDispatchBelowADInplaceOrView> below(std::in_place);
    const Routers r(in, mask, given, c);
    const at::Device device = r.logits[0].device();
    const c10::DeviceGuard guard(device);
    Tensor given_counts;
    if (counts_in) {
        TORCH_CHECK_TYPE(counts_in->scalar_type() == at::kLong && counts_in->device() == device,
                         "counts must be an int64 tensor on the device of the router logits");
        TORCH_CHECK_VALUE(counts_in->sizes() == at::IntArrayRef(c.shape(true)), "counts must be ", at::IntArrayRef(c.shape(true)), ", got ",
                          counts_in->sizes());
        given_counts = counts_in->contiguous();
    }
    const auto bytes = at::TensorOptions().dtype(at::kByte).device(device);
    const auto floats = bytes.dtype(at::kFloat);
    Tensor balance = at::empty(c.shape(false), floats), z = sigmoid ? Tensor() : at::empty(c.shape(false), floats);
    Tensor counts = at::empty(c.shape(true), bytes.dtype(at::kLong));
    Tensor kept = at::empty({c.groups() * (c.E + 1)}, floats);
    std::vector<DmRouterSet> sets(in.size());
    for (size_t i = 0; i < in.size(); ++i) describe(sets, i, r.logits[i], r.masks[i], r.experts[i], nullptr);
    const Tensor workspace = workspace_for(sets, c, bytes);
    float *slope = kept.mutable_data_ptr<float>();
    check(g.balance_loss(sets.data(), static_cast<int>(c.S), static_cast<int>(c.B), static_cast<int>(c.E), static_cast<int>(top_k), c.dtype,
                         c.sigmoid, c.per_image, given_counts.defined() ? given_counts.const_data_ptr<int64_t>() : nullptr,
                         balance.mutable_data_ptr<float>(), sigmoid ? nullptr : z.mutable_data_ptr<float>(),
                         counts.mutable_data_ptr<int64_t>(), slope, slope + c.groups() * c.E, workspace.mutable_data_ptr(),
                         workspace.numel(), status.mutable_data_ptr<int32_t>(), current_stream(device)),
          "dm_balance_loss");
    if (grad) {
        below.reset();                                 // (saving may run hooks)
        node->call = c;
        node->kept = Saved(kept);
        node->logits.resize(in.size());
        node->masked.resize(in.size());
        node->masks.resize(in.size());
        for (size_t i = 0; i < in.size(); ++i) {
            if (!in[i].requires_grad()) continue;
            node->logits[i] = Saved(r.logits[i]);
            node->masked[i] = r.masks[i].defined();
            if (node->masked[i]) node->masks[i] = Saved(r.masks[i]);
        }
        torch::autograd::set_history(balance, node);
        if (!sigmoid) torch::autograd::set_history(z, node);
    }
    return {balance, sigmoid ? std::nullopt : std::optional<Tensor>(z), counts};
}

Tensor expert_counts(const std::vector<Tensor> &in, int64_t top_k, const OptionalTensors &mask, bool per_image, const Tensor &status)
{
    RouterCall c{};
    c.top_k = top_k;
    c.per_image = per_image;
    refuse_tracing();
    const at::AutoDispatchBelowADInplaceOrView below;
    const Routers r(in, mask, OptionalTensors(in.size()), c);
    const at::Device device = r.logits[0].device();
    const c10::DeviceGuard guard(device);
    const auto bytes = at::TensorOptions().dtype(at::kByte).device(device);
    Tensor counts = at::empty(c.shape(true), bytes.dtype(at::kLong));
    std::vector<DmRouterSet> sets(in.size());
    for (size_t i = 0; i < in.size(); ++i) describe(sets, i, r.logits[i], r.masks[i], Tensor(), nullptr);
    const Tensor workspace = workspace_for(sets, c, bytes);
    check(g.expert_counts(sets.data(), static_cast<int>(c.S), static_cast<int>(c.B), static_cast<int>(c.E), static_cast<int>(top_k), c.dtype,
                          c.per_image, counts.mutable_data_ptr<int64_t>(), workspace.mutable_data_ptr(), workspace.numel(),
                          status.mutable_data_ptr<int32_t>(), current_stream(device)),
          "dm_expert_counts");
    return counts;
}

}  // namespace

extern "C" const char dm_loss_nodes_stamp[] = "detr_amd_loss_nodes built for torch " DM_BUILT_FOR_TORCH ";";

PYBIND11_MODULE(_loss_nodes, m)
{
    m.attr("built_for_torch") = DM_BUILT_FOR_TORCH;
    m.def("bind", torch::wrap_pybind_function(&bind));
    m.def("focal_losses", torch::wrap_pybind_function(&focal_losses));
    m.def("cross_entropies", torch::wrap_pybind_function(&cross_entropies));
    m.def("balance_losses", torch::wrap_pybind_function(&balance_losses));
    m.def("expert_counts", torch::wrap_pybind_function(&expert_counts));
    m.def("zero_word_outside_capture", torch::wrap_pybind_function(&zero_word_outside_capture));
}
