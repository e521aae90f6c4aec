// Compiled PyTorch binding of the operators around the attention: argument checks, output allocation, device guard and the
// C-ABI calls, as dispatcher operators of the `fpt_b200` library with their gradients.
//
//   fpt_b200::qk_rope            norm of every head and rotation, or the rotation alone (fpt_qk_rope)
//   fpt_b200::qk_norm_rope_bwd   gradient of the form with the norm
//   fpt_b200::linear_act         act(x W^T + b) + r (fpt_linear)
//   fpt_b200::linear_act_slope   the same with 2^15 act' in fp16 beside it, what a training step keeps
//   fpt_b200::linear_act_bwd     its gradient (fpt_linear_grad_act, _grad_input, _grad_weight)
//
// The Python module enters through plain functions that check the arguments that are not tensors and call the dispatcher
// (an eager call costs no boxing); graphs use torch.ops.fpt_b200.  Gradients are registered here as well: the backward
// pass of a small call is then a few microseconds of host time.  They are not themselves differentiable and say so.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>
#include <torch/library.h>

#include <cmath>
#include <cstring>
#include <memory>
#include <mutex>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/fpt_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kMaxHeadDim = 256, kMaxAxes = 4;

void check_status(int status, const char* entry) {
    TORCH_CHECK(status == 0, entry, " failed with status ", status, ": ", fpt_status_string(status));
}

fpt_stream_t stream_of(const Tensor& x) {
    return reinterpret_cast<fpt_stream_t>(at::cuda::getCurrentCUDAStream(x.device().index()).stream());
}

int dtype_id(at::ScalarType t) { return t == at::kFloat ? FPT_FP32 : t == at::kBFloat16 ? FPT_BF16 : FPT_FP16; }

bool floating(const Tensor& x) {
    return x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat;
}

// Gradients are not themselves differentiable.  Where autograd records the backward pass (create_graph) it is refused.  The
// transforms of torch.func always record it, also for a first derivative: there the gradients come back with a node that
// refuses when a second derivative reaches it.
[[noreturn]] void no_second_gradient(const char* name) {
    TORCH_CHECK(false, name, " has no second gradient: run its backward pass without create_graph");
}
bool of_transform(const Tensor& t) { return t.defined() && t.key_set().has(c10::DispatchKey::FuncTorchGradWrapper); }
// whether a transform records this backward pass
template <class... T>
bool in_transform(const char* name, const T&... tensors) {
    if (!at::GradMode::is_enabled()) return false;
    if (!c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) && !(of_transform(tensors) || ...))
        no_second_gradient(name);
    return true;
}
struct NoSecondGradient : torch::autograd::Node {
    const char* operator_name;
    explicit NoSecondGradient(const char* of) : operator_name(of) {}
    std::string name() const override { return "NoSecondGradient"; }
    torch::autograd::variable_list apply(torch::autograd::variable_list&&) override { no_second_gradient(operator_name); }
};
template <class... T>
void refuse_to_go_on(const char* name, std::initializer_list<Tensor> results, const T&... of) {
    if (!torch::autograd::compute_requires_grad(of...)) return;
    std::shared_ptr<NoSecondGradient> node(new NoSecondGradient(name), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(of...));
    for (const Tensor& t : results) torch::autograd::set_history(t, node);
}
// No keys of autograd on the way to the kernels, which spares host time, unless the backward pass is itself recorded.
struct BelowAutograd {
    std::optional<at::AutoDispatchBelowADInplaceOrView> guard;
    explicit BelowAutograd(bool recorded) {
        if (!recorded) guard.emplace();
    }
};

// a tangent would be lost below the autograd keys
template <class... T>
void no_forward_gradient(const char* name, const T&... inputs) {
    if (!torch::autograd::ForwardADLevel::try_get_by_idx(0)) return;      // no tangents anywhere: one look in place of one a tensor
    TORCH_CHECK(!((inputs.defined() && inputs._fw_grad(/*level=*/0).defined()) || ...), name, " has no forward-mode derivative");
}

// ---- fpt_qk_rope --------------------------------------------------------------------------------------------------

// the axis of every pair: the sections after one another (order 0), or dealt out in turn until an axis has its share (1)
std::vector<uint8_t> pair_axes(at::IntArrayRef sections, int64_t order) {
    std::vector<uint8_t> axes;
    if (order == 0) {
        for (size_t a = 0; a < sections.size(); ++a) axes.insert(axes.end(), size_t(sections[a]), uint8_t(a));
        return axes;
    }
    std::vector<int64_t> left(sections.begin(), sections.end());
    for (bool some = true; some;) {
        some = false;
        for (size_t a = 0; a < left.size(); ++a)
            if (left[a] > 0) {
                --left[a];
                axes.push_back(uint8_t(a));
                some = true;
            }
    }
    return axes;
}

struct Rope {
    int64_t batch, seq, q_heads, k_heads, dim, pairs;
    int position_bits = 0;
    int64_t pos_strides[3] = {0, 0, 0};
    std::vector<uint8_t> axes;
    int weight_dtype = FPT_FP32;
};

// Every check of a call, the devices last: what is wrong with shapes and types is said without a GPU as well.
Rope check_rope(const Tensor& q, const Tensor& k, const OptTensor& q_weight, const OptTensor& k_weight, const Tensor& increments,
                const OptTensor& positions, at::IntArrayRef sections, int64_t order, int64_t pairing, bool norm, double eps) {
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4, "q and k must have shape [batch, sequence, heads, head_dim]");
    TORCH_CHECK(floating(q), "q must be float16, bfloat16 or float32");
    TORCH_CHECK(q.scalar_type() == k.scalar_type(), "q and k must have the same dtype");
    TORCH_CHECK(q.size(0) == k.size(0), "q and k batch sizes must match");
    TORCH_CHECK(q.size(1) == k.size(1), "q and k sequence lengths must match");
    TORCH_CHECK(q.size(3) == k.size(3), "q and k head dimensions must match");
    TORCH_CHECK(q.size(2) > 0 && k.size(2) > 0, "q and k must contain at least one head");
    Rope r;
    r.batch = q.size(0), r.seq = q.size(1), r.q_heads = q.size(2), r.k_heads = k.size(2), r.dim = q.size(3);
    TORCH_CHECK(r.dim > 0 && r.dim % 8 == 0 && r.dim <= kMaxHeadDim, "head_dim must be a positive multiple of eight, at most ", kMaxHeadDim);
    TORCH_CHECK(increments.scalar_type() == at::kInt && increments.dim() == 1 && increments.is_contiguous(),
                "phase_increments must be a contiguous one-dimensional int32 tensor");
    r.pairs = increments.numel();
    TORCH_CHECK(r.pairs > 0 && r.pairs % 4 == 0 && 2 * r.pairs <= r.dim,
                "phase_increments must hold a positive multiple of four entries, at most head_dim / 2");
    TORCH_CHECK(pairing == FPT_PAIRS_ADJACENT || pairing == FPT_PAIRS_HALVES, "unknown pairing");
    TORCH_CHECK(order == 0 || order == 1, "unknown section order");
    for (const OptTensor* w : {&q_weight, &k_weight})
        if (w->has_value()) {
            TORCH_CHECK(norm, "weights go with the norm");
            TORCH_CHECK(floating(**w) && (*w)->dim() == 1 && (*w)->numel() == r.dim && (*w)->is_contiguous(),
                        "q_weight and k_weight must be contiguous float16, bfloat16 or float32 tensors of head_dim entries");
            r.weight_dtype = dtype_id((*w)->scalar_type());
        }
    TORCH_CHECK(!q_weight || !k_weight || q_weight->scalar_type() == k_weight->scalar_type(), "q_weight and k_weight must have the same dtype");
    TORCH_CHECK(!norm || (eps >= 0 && std::isfinite(float(eps))), "eps must be finite in fp32 and not negative");
    if (!sections.empty()) {
        TORCH_CHECK(positions.has_value(), "sections go with positions of one row per axis");
        TORCH_CHECK(int64_t(sections.size()) <= kMaxAxes, "at most ", kMaxAxes, " sections");
        int64_t sum = 0;
        for (int64_t n : sections) {
            TORCH_CHECK(n >= 0 && n <= r.pairs, "every section must hold between 0 and ", r.pairs, " pairs");
            sum += n;
        }
        TORCH_CHECK(sum == r.pairs, "the sections must add up to the ", r.pairs, " entries of phase_increments, got ", sum);
        r.axes = pair_axes(sections, order);
    }
    if (positions) {
        const Tensor& p = *positions;
        TORCH_CHECK(p.scalar_type() == at::kInt || p.scalar_type() == at::kLong, "positions must be int32 or int64");
        const int64_t lead = sections.empty() ? 0 : 1;
        TORCH_CHECK(p.dim() == lead + 1 || p.dim() == lead + 2, "positions must have shape ",
                    lead ? "[axes, sequence] or [axes, batch, sequence]" : "[sequence] or [batch, sequence]");
        TORCH_CHECK(!lead || p.size(0) == int64_t(sections.size()), "positions must have one row per section");
        TORCH_CHECK(p.size(-1) == r.seq, "positions must have the sequence length of q and k");
        const bool batched = p.dim() == lead + 2;
        TORCH_CHECK(!batched || p.size(lead) == r.batch || p.size(lead) == 1, "positions must have the batch size of q and k, or one row");
        r.position_bits = p.scalar_type() == at::kLong ? 64 : 32;
        r.pos_strides[0] = lead ? p.stride(0) : 0;
        r.pos_strides[1] = batched && p.size(lead) > 1 ? p.stride(lead) : 0;
        r.pos_strides[2] = p.stride(-1);
    }
    TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
    for (const Tensor& t : {k, increments, q_weight.value_or(q), k_weight.value_or(q), positions.value_or(q)})
        TORCH_CHECK(t.device() == q.device(), "all tensors must be on the CUDA device of q");
    return r;
}

// What the kernels take as it is: heads contiguous and on 16-byte boundaries, no more than 2 GB from a token's first to its
// last; anything else is copied.
Tensor rows_contiguous(const Tensor& t) {
    const int64_t item = t.element_size();
    bool fits = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int d = 0; d < 3; ++d) fits = fits && (t.size(d) < 2 || t.stride(d) * item % 16 == 0);
    fits = fits && (t.size(2) < 2 || t.stride(2) <= 0x7fffffff / item / t.size(2));
    return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

const void* pointer(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }

std::tuple<Tensor, Tensor> qk_rope(const Tensor& q_in, const Tensor& k_in, const OptTensor& q_weight, const OptTensor& k_weight,
                                   const Tensor& increments, const OptTensor& positions, at::IntArrayRef sections, int64_t order,
                                   int64_t pairing, bool norm, double eps, bool inverse) {
    const Rope r = check_rope(q_in, k_in, q_weight, k_weight, increments, positions, sections, order, pairing, norm, eps);
    TORCH_CHECK(!(norm && inverse), "inverse goes with the rotation alone");
    const c10::cuda::CUDAGuard guard(q_in.device());
    const Tensor q = rows_contiguous(q_in), k = rows_contiguous(k_in);
    Tensor q_out = at::empty(q.sizes(), q.options(), at::MemoryFormat::Contiguous);
    Tensor k_out = at::empty(k.sizes(), k.options(), at::MemoryFormat::Contiguous);
    check_status(fpt_qk_rope(q_out.data_ptr(), k_out.data_ptr(), q.data_ptr(), k.data_ptr(), pointer(q_weight), pointer(k_weight),
                             increments.data_ptr(), pointer(positions), r.position_bits, r.pos_strides,
                             r.axes.empty() ? nullptr : r.axes.data(), r.batch, r.seq, r.q_heads, r.k_heads, r.dim, r.pairs,
                             q.strides().data(), k.strides().data(), int(pairing), norm, float(eps), inverse,
                             dtype_id(q.scalar_type()), r.weight_dtype, stream_of(q)),
                 "fpt_qk_rope");
    return {q_out, k_out};
}

// weight gradients come back empty where they are not wanted
std::tuple<Tensor, Tensor, Tensor, Tensor> qk_norm_rope_bwd(const Tensor& dq_out_in, const Tensor& dk_out_in, const Tensor& q_in,
                                                            const Tensor& k_in, const OptTensor& q_weight, const OptTensor& k_weight,
                                                            const Tensor& increments, const OptTensor& positions,
                                                            at::IntArrayRef sections, int64_t order, int64_t pairing, double eps,
                                                            bool want_q_weight, bool want_k_weight) {
    const Rope r = check_rope(q_in, k_in, q_weight, k_weight, increments, positions, sections, order, pairing, true, eps);
    TORCH_CHECK(dq_out_in.sizes() == q_in.sizes() && dk_out_in.sizes() == k_in.sizes(), "gradients must have the shapes of q and k");
    TORCH_CHECK(dq_out_in.scalar_type() == q_in.scalar_type() && dk_out_in.scalar_type() == q_in.scalar_type(), "gradients must have the dtype of q and k");
    TORCH_CHECK(dq_out_in.device() == q_in.device() && dk_out_in.device() == q_in.device(), "gradients must be on the device of q");
    TORCH_CHECK((!want_q_weight || q_weight) && (!want_k_weight || k_weight), "a weight gradient goes with a weight");
    const c10::cuda::CUDAGuard guard(q_in.device());
    const Tensor q = rows_contiguous(q_in), k = rows_contiguous(k_in);
    const Tensor gq = rows_contiguous(dq_out_in), gk = rows_contiguous(dk_out_in);
    Tensor dq = at::empty(q.sizes(), q.options(), at::MemoryFormat::Contiguous);
    Tensor dk = at::empty(k.sizes(), k.options(), at::MemoryFormat::Contiguous);
    const auto options = (q_weight ? *q_weight : k_weight ? *k_weight : q).options();
    Tensor dqw = at::empty({want_q_weight ? r.dim : 0}, options), dkw = at::empty({want_k_weight ? r.dim : 0}, options);
    Tensor workspace;
    if (want_q_weight || want_k_weight)
        workspace = at::empty({fpt_qk_norm_rope_bwd_workspace_bytes(r.q_heads, r.k_heads, r.dim)}, q.options().dtype(at::kByte));
    check_status(fpt_qk_norm_rope_bwd(dq.data_ptr(), dk.data_ptr(), want_q_weight ? dqw.data_ptr() : nullptr,
                                      want_k_weight ? dkw.data_ptr() : nullptr, gq.data_ptr(), gk.data_ptr(), q.data_ptr(),
                                      k.data_ptr(), pointer(q_weight), pointer(k_weight), increments.data_ptr(), pointer(positions),
                                      r.position_bits, r.pos_strides, r.axes.empty() ? nullptr : r.axes.data(),
                                      workspace.defined() ? workspace.data_ptr() : nullptr, workspace.defined() ? workspace.numel() : 0,
                                      r.batch, r.seq, r.q_heads, r.k_heads, r.dim, r.pairs, q.strides().data(), k.strides().data(),
                                      gq.strides().data(), gk.strides().data(), int(pairing), float(eps),
                                      dtype_id(q.scalar_type()), r.weight_dtype, stream_of(q)),
                 "fpt_qk_norm_rope_bwd");
    return {dq, dk, dqw, dkw};
}

std::tuple<Tensor, Tensor> call_qk_rope(const Tensor& q, const Tensor& k, const OptTensor& q_weight, const OptTensor& k_weight,
                                        const Tensor& increments, const OptTensor& positions, at::IntArrayRef sections,
                                        int64_t order, int64_t pairing, bool norm, double eps, bool inverse) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("fpt_b200::qk_rope", "").typed<decltype(qk_rope)>();
    return op.call(q, k, q_weight, k_weight, increments, positions, sections, order, pairing, norm, eps, inverse);
}

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// a node like the generated ones of the library itself: a third of the host time of the generic custom function
struct QkRopeBackward : torch::autograd::Node {
    SavedVariable q, k, q_weight, k_weight, increments, positions;
    std::vector<int64_t> sections;
    int64_t order = 0, pairing = 0;
    bool norm = false, inverse = false, has_q_weight = false, has_k_weight = false, has_positions = false;
    double eps = 0;

    std::string name() const override { return "QkRopeBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable* v : {&q, &k, &q_weight, &k_weight, &increments, &positions}) v->reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(4);
        for (int i = 0; i < 2; ++i)
            if (!grads[i].defined()) grads[i] = input_metadata(i).zeros_like();
        // Everything is unpacked before the guard: a hook on a saved tensor (activation checkpointing) may run the forward pass
        // again, with its own graph.
        const OptTensor pos = has_positions ? OptTensor(positions.unpack()) : OptTensor();
        const Tensor inc = increments.unpack();
        if (!norm) {                    // the rotation alone needs neither q nor k again
            const BelowAutograd below(at::GradMode::is_enabled());      // linear: its gradient has one
            std::tie(out[0], out[1]) = call_qk_rope(grads[0], grads[1], {}, {}, inc, pos, sections, order, pairing, false, 0.0, !inverse);
            return out;
        }
        const Tensor q_in = q.unpack(), k_in = k.unpack();
        const OptTensor qw = has_q_weight ? OptTensor(q_weight.unpack()) : OptTensor(), kw = has_k_weight ? OptTensor(k_weight.unpack()) : OptTensor();
        static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("fpt_b200::qk_norm_rope_bwd", "").typed<decltype(qk_norm_rope_bwd)>();
        const bool dqw = has_q_weight && task_should_compute_output(2), dkw = has_k_weight && task_should_compute_output(3);
        const BelowAutograd below(in_transform("qk_rope", grads[0], grads[1], q_in, k_in, qw.value_or(Tensor()), kw.value_or(Tensor())));
        auto d = op.call(grads[0], grads[1], q_in, k_in, qw, kw, inc, pos, sections, order, pairing, eps, dqw, dkw);
        out[0] = std::get<0>(d);
        out[1] = std::get<1>(d);
        if (dqw) out[2] = std::get<2>(d);
        if (dkw) out[3] = std::get<3>(d);
        return out;
    }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> qk_norm_rope_bwd_autograd(const Tensor& dq_out, const Tensor& dk_out, const Tensor& q, const Tensor& k,
                                                                     const OptTensor& q_weight, const OptTensor& k_weight, const Tensor& increments,
                                                                     const OptTensor& positions, at::IntArrayRef sections, int64_t order,
                                                                     int64_t pairing, double eps, bool want_q_weight, bool want_k_weight) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("fpt_b200::qk_norm_rope_bwd", "").typed<decltype(qk_norm_rope_bwd)>();
    const Tensor qw = q_weight.value_or(Tensor()), kw = k_weight.value_or(Tensor());
    no_forward_gradient("qk_norm_rope_bwd", dq_out, dk_out, q, k, qw, kw);
    std::tuple<Tensor, Tensor, Tensor, Tensor> d;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        d = op.call(dq_out, dk_out, q, k, q_weight, k_weight, increments, positions, sections, order, pairing, eps, want_q_weight, want_k_weight);
    }
    refuse_to_go_on("qk_rope", {std::get<0>(d), std::get<1>(d), std::get<2>(d), std::get<3>(d)}, dq_out, dk_out, q, k, qw, kw);
    return d;
}

std::tuple<Tensor, Tensor> qk_rope_autograd(const Tensor& q, const Tensor& k, const OptTensor& q_weight, const OptTensor& k_weight,
                                            const Tensor& increments, const OptTensor& positions, at::IntArrayRef sections,
                                            int64_t order, int64_t pairing, bool norm, double eps, bool inverse) {
    const Tensor qw = q_weight.value_or(Tensor()), kw = k_weight.value_or(Tensor());
    no_forward_gradient("qk_rope", q, k, qw, kw);
    std::shared_ptr<QkRopeBackward> node;
    if (torch::autograd::compute_requires_grad(q, k, qw, kw)) {
        node = std::shared_ptr<QkRopeBackward>(new QkRopeBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(q, k, qw, kw));
        if (norm) {
            node->q = SavedVariable(q, false);
            node->k = SavedVariable(k, false);
        }
        node->has_q_weight = qw.defined();
        node->has_k_weight = kw.defined();
        if (qw.defined()) node->q_weight = SavedVariable(qw, false);
        if (kw.defined()) node->k_weight = SavedVariable(kw, false);
        node->increments = SavedVariable(increments, false);
        node->has_positions = positions.has_value();
        if (positions) node->positions = SavedVariable(*positions, false);
        node->sections = sections.vec();
        node->order = order, node->pairing = pairing, node->norm = norm, node->eps = eps, node->inverse = inverse;
    }
    std::tuple<Tensor, Tensor> out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        out = call_qk_rope(q, k, q_weight, k_weight, increments, positions, sections, order, pairing, norm, eps, inverse);
    }
    if (node) {
        torch::autograd::set_history(std::get<0>(out), node);
        torch::autograd::set_history(std::get<1>(out), node);
    }
    return out;
}

// ---- fpt_linear -----------------------------------------------------------------------------------------------------

// The word a bounded device-side wait reports to: mapped host memory, so that a call looks at it without a copy or an
// event.  One for each device, made together at the first call (also inside a stream capture, where plain allocation is an
// error).
constexpr int kMaxDevices = 64, kStatusBytes = 64;
volatile uint32_t* status_word(int64_t device) {
    static char* words = [] {
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        cudaThreadExchangeStreamCaptureMode(&mode);
        void* p = nullptr;
        const cudaError_t e = cudaHostAlloc(&p, kMaxDevices * kStatusBytes, cudaHostAllocPortable | cudaHostAllocMapped);
        cudaThreadExchangeStreamCaptureMode(&mode);
        TORCH_CHECK(e == cudaSuccess, "no host memory for the status words: ", cudaGetErrorString(e));
        std::memset(p, 0, kMaxDevices * kStatusBytes);
        return static_cast<char*>(p);
    }();
    TORCH_CHECK(device >= 0 && device < kMaxDevices, "no status word for device ", device);
    return reinterpret_cast<uint32_t*>(words + device * kStatusBytes);
}

void poll_linear_status(int64_t device) {
    volatile uint32_t* word = status_word(device);
    const uint32_t value = *word;
    if (value) {
        *word = 0;
        TORCH_CHECK(false, fpt_status_string(FPT_ERR_DEVICE_TIMEOUT), ": status word ", value, " (waiting point ", value & 0xffff,
                    ") left by an earlier linear_act on cuda:", device, "; the outputs of that call are invalid");
    }
}

struct Linear {
    int64_t rows, dim, out;
    std::vector<int64_t> shape;         // of the result
};

Linear check_linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, int64_t function,
                    int64_t degree, int64_t source) {
    TORCH_CHECK(x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16, "x must be float16 or bfloat16");
    TORCH_CHECK(weight.scalar_type() == x.scalar_type(), "x and weight must have the same dtype");
    TORCH_CHECK(x.dim() >= 1 && weight.dim() == 2, "x must be [..., dim] and weight [out, dim]");
    Linear l;
    l.dim = weight.size(1), l.out = weight.size(0);
    TORCH_CHECK(x.size(-1) == l.dim, "x has ", x.size(-1), " columns, the weight wants ", l.dim);
    TORCH_CHECK(l.dim > 0 && l.dim % 8 == 0, "dim must be a positive multiple of 8");
    TORCH_CHECK(l.out > 0, "weight must have at least one row");
    l.rows = x.numel() / l.dim;
    l.shape = x.sizes().vec();
    l.shape.back() = l.out;
    if (bias)
        TORCH_CHECK(floating(*bias) && bias->dim() == 1 && bias->numel() == l.out, "bias must be a float16, bfloat16 or float32 tensor of ", l.out, " entries");
    if (residual) {
        TORCH_CHECK(residual->scalar_type() == x.scalar_type(), "x and residual must have the same dtype");
        TORCH_CHECK(residual->sizes() == at::IntArrayRef(l.shape), "residual must have the shape of the result");
    }
    TORCH_CHECK(function >= FPT_FN_NONE && function <= FPT_FN_GELU && function != FPT_FN_ERF, "unknown activation");
    TORCH_CHECK(degree == 0 || (degree >= 3 && degree <= 6 && function != FPT_FN_NONE), "Unsupported degree: ", degree);
    TORCH_CHECK(source == 0 || (source == 1 && x.scalar_type() == at::kBFloat16), "FP16 spline kernels only support coeff_source=current");
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    for (const Tensor& t : {weight, bias.value_or(x), residual.value_or(x)})
        TORCH_CHECK(t.device() == x.device(), "all tensors must be on the CUDA device of x");
    return l;
}

int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// [rows, columns] with contiguous rows that do not overlap
Tensor as_rows(const Tensor& t, int64_t rows, int64_t columns) {
    Tensor r = t.reshape({rows, columns});
    if ((columns > 1 && r.stride(1) != 1) || (rows > 1 && r.stride(0) < columns)) r = r.contiguous();
    return r;
}
bool loadable(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && row_stride(t) % 8 == 0; }
// the same as a matrix operand: rows on 16-byte boundaries
Tensor as_operand(const Tensor& t, int64_t rows, int64_t columns) {
    Tensor r = as_rows(t, rows, columns);
    return loadable(r) ? r : r.clone(at::MemoryFormat::Contiguous);
}

std::tuple<Tensor, Tensor> run_linear(const Tensor& x_in, const Tensor& weight_in, const OptTensor& bias_in, const OptTensor& residual_in,
                                      int64_t function, int64_t degree, int64_t source, bool want_slope) {
    const Linear l = check_linear(x_in, weight_in, bias_in, residual_in, function, degree, source);
    const c10::cuda::CUDAGuard guard(x_in.device());
    poll_linear_status(x_in.device().index());
    Tensor out = at::empty(l.shape, x_in.options(), at::MemoryFormat::Contiguous);
    const int64_t padded = (l.out + 7) / 8 * 8;
    Tensor slope = at::empty({want_slope && function != FPT_FN_NONE ? l.rows : 0, padded}, x_in.options().dtype(at::kHalf), at::MemoryFormat::Contiguous);
    if (l.rows == 0) return {out, slope};
    const Tensor x = as_operand(x_in, l.rows, l.dim), weight = as_operand(weight_in, l.out, l.dim);
    const Tensor bias = bias_in ? bias_in->contiguous() : Tensor();
    const Tensor residual = residual_in ? as_rows(*residual_in, l.rows, l.out) : Tensor();
    const int rc = fpt_linear(out.data_ptr(), slope.numel() ? slope.data_ptr() : nullptr, x.data_ptr(), weight.data_ptr(),
                              bias.defined() ? bias.data_ptr() : nullptr, residual.defined() ? residual.data_ptr() : nullptr, l.rows,
                              l.dim, l.out, row_stride(x), row_stride(weight), l.out, residual.defined() ? row_stride(residual) : 0,
                              padded, dtype_id(x.scalar_type()), bias.defined() ? dtype_id(bias.scalar_type()) : FPT_FP32,
                              int(function), int(degree), int(source), const_cast<uint32_t*>(status_word(x.device().index())), stream_of(x));
    TORCH_CHECK(rc != FPT_ERR_UNKNOWN_PROGRAM, "Unsupported activation degree: ", degree);
    check_status(rc, "fpt_linear");
    return {out, slope};
}

Tensor linear_act(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, int64_t function,
                  int64_t degree, int64_t source) {
    return std::get<0>(run_linear(x, weight, bias, residual, function, degree, source, false));
}

std::tuple<Tensor, Tensor> linear_act_slope(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                                            int64_t function, int64_t degree, int64_t source) {
    return run_linear(x, weight, bias, residual, function, degree, source, true);
}

// dx, dW, db; empty where not wanted.  slope: empty for no activation.  bias_dtype: 0 float16, 1 bfloat16, 2 float32.
std::tuple<Tensor, Tensor, Tensor> linear_act_bwd(const Tensor& dy_in, const Tensor& slope, const OptTensor& x_in, const OptTensor& weight_in,
                                                  at::IntArrayRef x_shape, int64_t out, int64_t bias_dtype, bool want_x, bool want_weight,
                                                  bool want_bias) {
    TORCH_CHECK(dy_in.is_cuda(), "the gradient must be a CUDA tensor");
    TORCH_CHECK(dy_in.scalar_type() == at::kHalf || dy_in.scalar_type() == at::kBFloat16, "the gradient must be float16 or bfloat16");
    TORCH_CHECK(!x_shape.empty() && out > 0 && dy_in.dim() == int64_t(x_shape.size()) && dy_in.size(-1) == out, "the gradient must have the shape of the result");
    TORCH_CHECK((!want_x || weight_in) && (!want_weight || x_in), "the weight and x are needed for each other's gradient");
    TORCH_CHECK(bias_dtype >= FPT_FP16 && bias_dtype <= FPT_FP32, "unknown bias dtype");
    const int64_t dim = x_shape.back(), rows = dy_in.numel() / out, padded = (out + 7) / 8 * 8;
    int64_t expected = 1;
    for (size_t i = 0; i + 1 < x_shape.size(); ++i) expected *= x_shape[i];
    TORCH_CHECK(rows == expected, "the gradient must have the shape of the result");
    TORCH_CHECK(slope.numel() == 0 || (slope.scalar_type() == at::kHalf && slope.is_contiguous() && slope.numel() == rows * padded &&
                                       slope.device() == dy_in.device()), "the slope does not fit the gradient");
    for (const OptTensor* t : {&x_in, &weight_in})
        if (t->has_value())
            TORCH_CHECK((*t)->scalar_type() == dy_in.scalar_type() && (*t)->device() == dy_in.device(), "x and weight must have the gradient's dtype and device");
    TORCH_CHECK(!want_x || (weight_in->dim() == 2 && weight_in->size(0) == out && weight_in->size(1) == dim), "the weight does not fit the gradient");
    TORCH_CHECK(!want_weight || x_in->sizes() == x_shape, "x does not fit the gradient");
    const c10::cuda::CUDAGuard guard(dy_in.device());
    poll_linear_status(dy_in.device().index());
    const int dtype = dtype_id(dy_in.scalar_type());
    Tensor dx = at::empty(want_x ? x_shape : at::IntArrayRef({0}), dy_in.options(), at::MemoryFormat::Contiguous);
    Tensor dw = at::empty({want_weight ? out : 0, dim}, dy_in.options(), at::MemoryFormat::Contiguous);
    Tensor db = at::empty({want_bias ? out : 0}, dy_in.options().dtype(bias_dtype == FPT_FP32 ? at::kFloat : bias_dtype == FPT_BF16 ? at::kBFloat16 : at::kHalf));
    const Tensor dy = rows ? as_rows(dy_in, rows, out) : dy_in.reshape({0, out});
    const bool products = want_x || want_weight;
    Tensor dz = dy;
    const bool copy = rows && products && (slope.numel() || !loadable(dy));
    if (copy) dz = at::empty({rows, padded}, dy.options(), at::MemoryFormat::Contiguous);
    if (copy || want_bias) {
        const int64_t bytes = want_bias ? fpt_linear_grad_act_workspace_bytes(rows, out) : 0;
        Tensor workspace = at::empty({bytes}, dy.options().dtype(at::kByte));
        check_status(fpt_linear_grad_act(copy ? dz.data_ptr() : nullptr, want_bias ? db.data_ptr() : nullptr, dy.data_ptr(),
                                         slope.numel() ? slope.data_ptr() : nullptr, bytes ? workspace.data_ptr() : nullptr, bytes, rows, out,
                                         padded, rows ? row_stride(dy) : out, padded, dtype, int(bias_dtype), stream_of(dy)),
                     "fpt_linear_grad_act");
    }
    void* status = const_cast<uint32_t*>(status_word(dy_in.device().index()));
    const int64_t dz_ld = copy ? padded : rows ? row_stride(dz) : padded;
    if (want_x && rows) {
        const Tensor weight = as_operand(*weight_in, out, dim);
        check_status(fpt_linear_grad_input(dx.data_ptr(), dz.data_ptr(), weight.data_ptr(), rows, dim, out, dim, dz_ld, row_stride(weight), dtype,
                                           status, stream_of(dy)),
                     "fpt_linear_grad_input");
    }
    if (want_weight) {
        const Tensor x = rows ? as_operand(*x_in, rows, dim) : *x_in;
        check_status(fpt_linear_grad_weight(dw.data_ptr(), dz.data_ptr(), x.data_ptr(), rows, dim, out, dim, dz_ld, rows ? row_stride(x) : dim, dtype,
                                            status, stream_of(dy)),
                     "fpt_linear_grad_weight");
    }
    return {dx, dw, db};
}

Tensor call_linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, int64_t function,
                   int64_t degree, int64_t source) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("fpt_b200::linear_act", "").typed<decltype(linear_act)>();
    return op.call(x, weight, bias, residual, function, degree, source);
}

// linear_act_bwd as the dispatcher knows it: sizes may be symbols of a compiled graph
using linear_act_bwd_symbolic = std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&,
                                                                   c10::SymIntArrayRef, c10::SymInt, int64_t, bool, bool, bool);

struct LinearBackward : torch::autograd::Node {
    SavedVariable x, weight, slope;
    std::vector<c10::SymInt> shape;     // of x
    c10::SymInt out = 0;
    int64_t bias_dtype = 0;
    bool has_bias = false;

    std::string name() const override { return "LinearActBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable* v : {&x, &weight, &slope}) v->reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list result(4);
        if (!grads[0].defined()) return result;
        const bool want_x = task_should_compute_output(0), want_w = task_should_compute_output(1), want_b = has_bias && task_should_compute_output(2);
        if (want_x || want_w || want_b) {
            static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("fpt_b200::linear_act_bwd", "").typed<linear_act_bwd_symbolic>();
            // unpacked before the guard, as above
            const Tensor kept = slope.unpack(), x_in = want_w ? x.unpack() : Tensor(), weight_in = want_x ? weight.unpack() : Tensor();
            const BelowAutograd below(in_transform("linear_act", grads[0], kept, x_in, weight_in));
            auto d = op.call(grads[0], kept, want_w ? OptTensor(x_in) : OptTensor(), want_x ? OptTensor(weight_in) : OptTensor(), shape, out,
                             bias_dtype, want_x, want_w, want_b);
            if (want_x) result[0] = std::get<0>(d);
            if (want_w) result[1] = std::get<1>(d);
            if (want_b) result[2] = std::get<2>(d);
        }
        if (task_should_compute_output(3)) result[3] = grads[0];
        return result;
    }
};

std::tuple<Tensor, Tensor, Tensor> linear_act_bwd_autograd(const Tensor& dy, const Tensor& slope, const OptTensor& x, const OptTensor& weight,
                                                           c10::SymIntArrayRef x_shape, c10::SymInt out, int64_t bias_dtype, bool want_x,
                                                           bool want_weight, bool want_bias) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("fpt_b200::linear_act_bwd", "").typed<linear_act_bwd_symbolic>();
    const Tensor xs = x.value_or(Tensor()), ws = weight.value_or(Tensor());
    no_forward_gradient("linear_act_bwd", dy, slope, xs, ws);
    std::tuple<Tensor, Tensor, Tensor> d;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        d = op.call(dy, slope, x, weight, x_shape, out, bias_dtype, want_x, want_weight, want_bias);
    }
    refuse_to_go_on("linear_act", {std::get<0>(d), std::get<1>(d), std::get<2>(d)}, dy, slope, xs, ws);
    return d;
}

// what a training step runs: the result with its node, and the slope (empty where nobody asks for it)
std::tuple<Tensor, Tensor> linear_recorded(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                                           int64_t function, int64_t degree, int64_t source, bool want_slope) {
    static const auto with_slope = c10::Dispatcher::singleton().findSchemaOrThrow("fpt_b200::linear_act_slope", "").typed<decltype(linear_act_slope)>();
    const Tensor b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
    no_forward_gradient("linear_act", x, weight, b, r);
    std::shared_ptr<LinearBackward> node;
    bool keep_slope = want_slope;       // no activation: the slope is 1; only the residual wants a gradient: nobody asks for it
    if (torch::autograd::compute_requires_grad(x, weight, b, r)) {
        node = std::shared_ptr<LinearBackward>(new LinearBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, weight, b, r));
        if (weight.requires_grad()) node->x = SavedVariable(x, false);
        if (x.requires_grad()) node->weight = SavedVariable(weight, false);
        node->shape = x.sym_sizes().vec();
        node->out = weight.dim() ? weight.sym_size(0) : c10::SymInt(0);
        node->has_bias = b.defined();
        node->bias_dtype = b.defined() ? dtype_id(b.scalar_type()) : FPT_FP32;
        keep_slope |= function != FPT_FN_NONE && (x.requires_grad() || weight.requires_grad() || (b.defined() && b.requires_grad()));
    }
    Tensor out, slope;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        if (keep_slope) std::tie(out, slope) = with_slope.call(x, weight, bias, residual, function, degree, source);
        else out = call_linear(x, weight, bias, residual, function, degree, source);
        if (node && !keep_slope) slope = out.new_empty({0, 8}, at::TensorOptions().dtype(at::kHalf));
    }
    if (node) {
        node->slope = SavedVariable(slope, false);
        torch::autograd::set_history(out, node);
    }
    return {out, slope};
}

Tensor linear_autograd(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, int64_t function,
                       int64_t degree, int64_t source) {
    return std::get<0>(linear_recorded(x, weight, bias, residual, function, degree, source, false));
}

std::tuple<Tensor, Tensor> linear_slope_autograd(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                                                 int64_t function, int64_t degree, int64_t source) {
    auto both = linear_recorded(x, weight, bias, residual, function, degree, source, true);
    refuse_to_go_on("linear_act", {std::get<1>(both)}, x, weight, bias.value_or(Tensor()), residual.value_or(Tensor()));
    return both;
}

// the eager doors: off the GPU the checks run here, where no kernel would be found
Tensor enter_linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, int64_t function,
                    int64_t degree, int64_t source) {
    if (!x.is_cuda()) check_linear(x, weight, bias, residual, function, degree, source);
    return call_linear(x, weight, bias, residual, function, degree, source);
}

std::tuple<Tensor, Tensor> enter_qk_rope(const Tensor& q, const Tensor& k, const OptTensor& q_weight, const OptTensor& k_weight,
                                         const Tensor& increments, const OptTensor& positions, const std::vector<int64_t>& sections,
                                         int64_t order, int64_t pairing, bool norm, double eps) {
    if (!q.is_cuda() || !k.is_cuda()) check_rope(q, k, q_weight, k_weight, increments, positions, sections, order, pairing, norm, eps);
    return call_qk_rope(q, k, q_weight, k_weight, increments, positions, sections, order, pairing, norm, eps, false);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(fpt_b200, m) {
    m.def("qk_rope(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor phase_increments, Tensor? positions, "
          "int[] sections, int section_order, int pairing, bool norm, float eps, bool inverse) -> (Tensor, Tensor)");
    m.def("qk_norm_rope_bwd(Tensor dq_out, Tensor dk_out, Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, "
          "Tensor phase_increments, Tensor? positions, int[] sections, int section_order, int pairing, float eps, "
          "bool want_q_weight, bool want_k_weight) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("linear_act(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int function, int degree, int source) -> Tensor");
    m.def("linear_act_slope(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int function, int degree, int source) -> (Tensor, Tensor)");
    m.def("linear_act_bwd(Tensor dy, Tensor slope, Tensor? x, Tensor? weight, SymInt[] x_shape, SymInt out, int bias_dtype, bool want_x, "
          "bool want_weight, bool want_bias) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(fpt_b200, CUDA, m) {
    m.impl("qk_rope", &qk_rope);
    m.impl("qk_norm_rope_bwd", &qk_norm_rope_bwd);
    m.impl("linear_act", &linear_act);
    m.impl("linear_act_slope", &linear_act_slope);
    m.impl("linear_act_bwd", &linear_act_bwd);
}

TORCH_LIBRARY_IMPL(fpt_b200, Autograd, m) {
    m.impl("qk_rope", &qk_rope_autograd);
    m.impl("qk_norm_rope_bwd", &qk_norm_rope_bwd_autograd);
    m.impl("linear_act", &linear_autograd);
    m.impl("linear_act_slope", &linear_slope_autograd);
    m.impl("linear_act_bwd", &linear_act_bwd_autograd);
}

void register_block_operators(pybind11::module_& m) {
    m.def("qk_rope", &enter_qk_rope);
    m.def("linear_act", &enter_linear);
    m.def("poll_linear_status", &poll_linear_status);
    m.def("linear_status_address", [](int64_t device) { return reinterpret_cast<uintptr_t>(status_word(device)); });
}
