// Compiled PyTorch binding of the operators around the attention: argument checks, output allocation, device guard and the
// C-ABI calls, as dispatcher operators of the `fpt_b200` library with their gradients.
//
//   fpt_b200::qk_rope            norm of every head and rotation, or the rotation alone (fpt_qk_rope)
//   fpt_b200::qk_norm_rope_bwd   gradient of the form with the norm
//
// The Python module enters through plain functions that check the arguments that are not tensors and call the dispatcher
// (an eager call costs no boxing); graphs use torch.ops.fpt_b200.  Gradients are registered here as well: the backward
// pass of a small call is then a few microseconds of host time.  They are not themselves differentiable and say so.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/extension.h>
#include <torch/library.h>

#include <cmath>
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

void no_second_gradient(const char* name) {
    TORCH_CHECK(!at::GradMode::is_enabled(), name, " has no second gradient: run its backward pass without create_graph");
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
    TORCH_CHECK(!norm || (eps >= 0 && std::isfinite(eps)), "eps must be finite and not negative");
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

Tensor rows_contiguous(const Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }

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

struct QkRopeFunction : torch::autograd::Function<QkRopeFunction> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k,
                                                  const OptTensor& q_weight, const OptTensor& k_weight, const Tensor& increments,
                                                  const OptTensor& positions, std::vector<int64_t> sections, int64_t order,
                                                  int64_t pairing, bool norm, double eps, bool inverse) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto out = call_qk_rope(q, k, q_weight, k_weight, increments, positions, sections, order, pairing, norm, eps, inverse);
        // the rotation alone needs neither q nor k again
        ctx->save_for_backward({norm ? q : Tensor(), norm ? k : Tensor(), q_weight.value_or(Tensor()), k_weight.value_or(Tensor()),
                                increments, positions.value_or(Tensor())});
        ctx->saved_data["sections"] = sections;
        ctx->saved_data["order"] = order;
        ctx->saved_data["pairing"] = pairing;
        ctx->saved_data["norm"] = norm;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["inverse"] = inverse;
        ctx->saved_data["dq_weight"] = q_weight.has_value() && q_weight->requires_grad();
        ctx->saved_data["dk_weight"] = k_weight.has_value() && k_weight->requires_grad();
        return {std::get<0>(out), std::get<1>(out)};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        no_second_gradient("qk_rope");
        const auto saved = ctx->get_saved_variables();
        const auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
        const auto sections = ctx->saved_data["sections"].toIntVector();
        const int64_t order = ctx->saved_data["order"].toInt(), pairing = ctx->saved_data["pairing"].toInt();
        torch::autograd::variable_list out(12);
        if (!ctx->saved_data["norm"].toBool()) {
            std::tie(out[0], out[1]) = call_qk_rope(grads[0], grads[1], {}, {}, saved[4], opt(saved[5]), sections, order, pairing,
                                                    false, 0.0, !ctx->saved_data["inverse"].toBool());
            return out;
        }
        static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("fpt_b200::qk_norm_rope_bwd", "").typed<decltype(qk_norm_rope_bwd)>();
        const bool dqw = ctx->saved_data["dq_weight"].toBool(), dkw = ctx->saved_data["dk_weight"].toBool();
        auto d = op.call(grads[0], grads[1], saved[0], saved[1], opt(saved[2]), opt(saved[3]), saved[4], opt(saved[5]), sections, order,
                         pairing, ctx->saved_data["eps"].toDouble(), dqw, dkw);
        out[0] = std::get<0>(d);
        out[1] = std::get<1>(d);
        if (dqw) out[2] = std::get<2>(d);
        if (dkw) out[3] = std::get<3>(d);
        return out;
    }
};

std::tuple<Tensor, Tensor> qk_rope_autograd(const Tensor& q, const Tensor& k, const OptTensor& q_weight, const OptTensor& k_weight,
                                            const Tensor& increments, const OptTensor& positions, at::IntArrayRef sections,
                                            int64_t order, int64_t pairing, bool norm, double eps, bool inverse) {
    const bool wanted = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || (q_weight && q_weight->requires_grad()) ||
                                                       (k_weight && k_weight->requires_grad()));
    if (!wanted) {
        at::AutoDispatchBelowADInplaceOrView below;
        return call_qk_rope(q, k, q_weight, k_weight, increments, positions, sections, order, pairing, norm, eps, inverse);
    }
    auto out = QkRopeFunction::apply(q, k, q_weight, k_weight, increments, positions, sections.vec(), order, pairing, norm, eps, inverse);
    return {out[0], out[1]};
}

// the eager door: off the GPU the checks run here, where no kernel would be found
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
}

TORCH_LIBRARY_IMPL(fpt_b200, CUDA, m) {
    m.impl("qk_rope", &qk_rope);
    m.impl("qk_norm_rope_bwd", &qk_norm_rope_bwd);
}

TORCH_LIBRARY_IMPL(fpt_b200, Autograd, m) {
    m.impl("qk_rope", &qk_rope_autograd);
}

void register_block_operators(pybind11::module_& m) {
    m.def("qk_rope", &enter_qk_rope);
}
