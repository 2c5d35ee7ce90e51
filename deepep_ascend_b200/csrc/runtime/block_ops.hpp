// Tensor front end of the operators around the expert layer: argument checks, result tensors, launches on the current stream.
#pragma once
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <optional>
#include <tuple>
#include <vector>

#include "../kernels/api.h"
#include "elastic_buffer.hpp"

namespace ep_host {

// Whether something records, transforms or intercepts what is done with these tensors, or a tangent goes with one of them: a native call would be invisible to it (a tracer would
// record the allocation of the results and not the launch that fills them).  Asked here since it takes a tenth of the time that the same questions take in Python.
inline bool watched(std::initializer_list<const at::Tensor*> tensors) {
    if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::stack_len() != 0 ||
        c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode))
        return true;
    constexpr c10::DispatchKeySet kWrappers({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::Functionalize});
    for (const at::Tensor* t : tensors)
        if (t != nullptr && t->defined() && (t->key_set().has_any(kWrappers) || t->_fw_grad(0).defined())) return true;
    return false;
}
// ... or a gradient is to be carried on through one of them
inline bool not_for_a_kernel(std::initializer_list<const at::Tensor*> tensors) {
    if (at::GradMode::is_enabled())
        for (const at::Tensor* t : tensors)
            if (t != nullptr && t->requires_grad()) return true;
    return watched(tensors);
}
inline const at::Tensor* given(const std::optional<at::Tensor>& t) { return t.has_value() ? &*t : nullptr; }

inline int device_sms() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }

// A contiguous tensor on a part of `bytes`, an allocation that several results of one call share: making them one by one is a fifth of the time of a small call
inline at::Tensor part_of(const at::Tensor& bytes, int64_t offset, at::IntArrayRef sizes, at::ScalarType type) {
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(bytes.storage()), bytes.key_set(), c10::scalarTypeToTypeMeta(type));
    impl->set_storage_offset(offset / static_cast<int64_t>(c10::elementSize(type)));
    impl->set_sizes_contiguous(sizes);
    return at::Tensor(std::move(impl));
}
inline int64_t round16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

inline void router_logits(RouterArgs& a, const at::Tensor& logits) {
    TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16),
                "logits must be fp32 or bf16 [tokens, experts] on a GPU");
    TORCH_CHECK(logits.size(1) >= 1 && logits.size(1) <= EP_MAX_EXPERTS, "between 1 and ", EP_MAX_EXPERTS, " experts");
    TORCH_CHECK(logits.size(1) == 1 || logits.stride(1) == 1, "rows of the logits must be contiguous");
    TORCH_CHECK(logits.size(0) <= 1 || logits.stride(0) >= logits.size(1), "rows of the logits must not overlap");
    TORCH_CHECK(logits.size(0) < (1ll << 31), "too many tokens");
    a.logits = logits.data_ptr();
    a.ld = std::max(logits.stride(0), logits.size(1));
    a.logits_bf16 = logits.scalar_type() == at::kBFloat16;
    a.num_tokens = static_cast<int>(logits.size(0));
    a.num_experts = static_cast<int>(logits.size(1));
}

// (nothing where a kernel is not to run, as of the norm below)
using Routes = std::tuple<at::Tensor, at::Tensor, at::Tensor>;
inline std::optional<Routes> route(const at::Tensor& logits, int64_t num_topk, bool softmax, const std::optional<at::Tensor>& bias, int64_t num_groups, int64_t num_topk_groups,
                                   int64_t group_top, bool renormalize, double scale, const std::optional<at::Tensor>& token_mask, bool idx_is_64) {
    if (not_for_a_kernel({&logits}) || watched({given(bias), given(token_mask)})) return std::nullopt;      // (the bias, which the choice alone sees, has no gradient)
    RouterArgs a{};
    router_logits(a, logits);
    TORCH_CHECK(num_groups >= 1 && num_groups <= 32 && a.num_experts % num_groups == 0, "the experts must divide into 1 to 32 groups");
    TORCH_CHECK(num_topk_groups >= 1 && num_topk_groups <= num_groups, "num_topk_groups must be between 1 and num_groups");
    TORCH_CHECK(num_topk >= 1 && num_topk <= EP_MAX_TOPK && num_topk <= a.num_experts / num_groups * num_topk_groups,
                "num_topk must be between 1 and ", EP_MAX_TOPK, ", and at most the experts of num_topk_groups groups");
    TORCH_CHECK(num_groups == 1 || group_top == 1 || (group_top == 2 && a.num_experts / num_groups >= 2), "group_top must be 1 or 2, and at most the experts of a group");
    const c10::cuda::CUDAGuard guard(logits.device());
    if (bias.has_value()) {
        TORCH_CHECK(bias->device() == logits.device() && bias->scalar_type() == at::kFloat && bias->is_contiguous() && bias->dim() == 1 && bias->size(0) == a.num_experts,
                    "bias must be contiguous fp32 [experts] on the device of the logits");
        a.bias = bias->data_ptr<float>();
    }
    if (token_mask.has_value()) {
        TORCH_CHECK(token_mask->device() == logits.device() && token_mask->scalar_type() == at::kBool && token_mask->is_contiguous() && token_mask->dim() == 1 &&
                        token_mask->size(0) == a.num_tokens,
                    "token_mask must be contiguous bool [tokens] on the device of the logits");
        a.token_mask = reinterpret_cast<const uint8_t*>(token_mask->data_ptr<bool>());
    }
    const int64_t pairs = a.num_tokens * num_topk, idx_bytes = round16(pairs * (idx_is_64 ? 8 : 4)), weight_bytes = round16(pairs * 4);
    at::Tensor results = at::empty({idx_bytes + weight_bytes + 4 * a.num_experts}, logits.options().dtype(at::kByte));
    at::Tensor idx = part_of(results, 0, {a.num_tokens, num_topk}, idx_is_64 ? at::kLong : at::kInt);
    at::Tensor weights = part_of(results, idx_bytes, {a.num_tokens, num_topk}, at::kFloat);
    at::Tensor count = part_of(results, idx_bytes + weight_bytes, {a.num_experts}, at::kInt);
    a.num_topk = static_cast<int>(num_topk);
    a.softmax = softmax;
    a.renormalize = renormalize;
    a.scale = static_cast<float>(scale);
    a.num_groups = static_cast<int>(num_groups);
    a.num_topk_groups = static_cast<int>(num_topk_groups);
    a.group_top = static_cast<int>(num_groups == 1 ? 1 : group_top);
    a.topk_idx = idx.data_ptr();
    a.idx_is_64 = idx_is_64;
    a.topk_weights = weights.data_ptr<float>();
    a.count = count.data_ptr<int32_t>();
    cuda_check(ep::launch_route(a, device_sms(), at::cuda::getCurrentCUDAStream()), "routing launch");
    return Routes(idx, weights, count);
}

inline std::optional<at::Tensor> route_backward(const at::Tensor& d_weights, const at::Tensor& logits, const at::Tensor& topk_idx, bool softmax, bool renormalize, double scale) {
    if (not_for_a_kernel({&d_weights, &logits, &topk_idx})) return std::nullopt;
    RouterArgs a{};
    router_logits(a, logits);
    TORCH_CHECK(topk_idx.device() == logits.device() && topk_idx.dim() == 2 && topk_idx.is_contiguous() && topk_idx.size(0) == a.num_tokens &&
                    topk_idx.size(1) >= 1 && topk_idx.size(1) <= EP_MAX_TOPK && (topk_idx.scalar_type() == at::kLong || topk_idx.scalar_type() == at::kInt),
                "topk_idx must be contiguous int64 or int32 [tokens, K] on the device of the logits, K at most ", EP_MAX_TOPK);
    TORCH_CHECK(d_weights.device() == logits.device() && d_weights.scalar_type() == at::kFloat && d_weights.is_contiguous() && d_weights.sizes() == topk_idx.sizes(),
                "d_weights must be contiguous fp32 of topk_idx's shape on the device of the logits");
    const c10::cuda::CUDAGuard guard(logits.device());
    at::Tensor d_logits = at::empty({a.num_tokens, a.num_experts}, logits.options());
    a.num_topk = static_cast<int>(topk_idx.size(1));
    a.softmax = softmax;
    a.renormalize = renormalize;
    a.scale = static_cast<float>(scale);
    a.topk_idx = topk_idx.data_ptr();
    a.idx_is_64 = topk_idx.scalar_type() == at::kLong;
    a.d_weights = d_weights.data_ptr<float>();
    a.d_logits = d_logits.data_ptr();
    cuda_check(ep::launch_route_backward(a, device_sms(), at::cuda::getCurrentCUDAStream()), "routing gradient launch");
    return d_logits;
}

inline bool is_bf16_or_f32(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }

inline void norm_rows(LayerNormArgs& a, const at::Tensor& x, const at::Tensor& weight) {
    TORCH_CHECK(x.is_cuda() && x.dim() == 2 && is_bf16_or_f32(x), "x must be bf16 or fp32 [rows, hidden] on a GPU");
    TORCH_CHECK(x.size(1) >= 1 && x.size(1) < (1ll << 24) && x.size(0) < (1ll << 31), "between 1 and 2^24 - 1 channels, fewer than 2^31 rows");
    TORCH_CHECK(x.size(1) == 1 || x.stride(1) == 1, "rows of x must be contiguous");
    TORCH_CHECK(weight.device() == x.device() && is_bf16_or_f32(weight) && weight.is_contiguous() && weight.dim() == 1 && weight.size(0) == x.size(1),
                "weight must be contiguous bf16 or fp32 [hidden] on the device of x");
    a.x = x.data_ptr();
    a.ldx = x.stride(0);
    a.rows = static_cast<int>(x.size(0));
    a.hidden = static_cast<int>(x.size(1));
    a.x_bf16 = x.scalar_type() == at::kBFloat16;
    a.param_bf16 = weight.scalar_type() == at::kBFloat16;
    a.weight = weight.data_ptr();
}

// nothing: for the PyTorch statement, or the function that carries gradients
using NormResults = std::tuple<at::Tensor, at::Tensor, at::Tensor>;
inline std::optional<NormResults> layer_norm(const at::Tensor& x, const at::Tensor& weight, const std::optional<at::Tensor>& bias, double eps) {
    if (not_for_a_kernel({&x, &weight, given(bias)})) return std::nullopt;
    LayerNormArgs a{};
    norm_rows(a, x, weight);
    if (bias.has_value()) {
        TORCH_CHECK(bias->device() == x.device() && bias->scalar_type() == weight.scalar_type() && bias->is_contiguous() && bias->sizes() == weight.sizes(),
                    "bias must be like the weight");
        a.bias = bias->data_ptr();
    }
    const c10::cuda::CUDAGuard guard(x.device());
    at::Tensor y = at::empty({x.size(0), x.size(1)}, x.options());
    at::Tensor moments = at::empty({2 * round16(4 * x.size(0))}, x.options().dtype(at::kByte));
    at::Tensor mean = part_of(moments, 0, {x.size(0)}, at::kFloat), rstd = part_of(moments, round16(4 * x.size(0)), {x.size(0)}, at::kFloat);
    a.eps = static_cast<float>(eps);
    a.y = y.data_ptr();
    a.mean = mean.data_ptr<float>();
    a.rstd = rstd.data_ptr<float>();
    cuda_check(ep::launch_layer_norm(a, device_sms(), at::cuda::getCurrentCUDAStream()), "layer norm launch");
    return NormResults(y, mean, rstd);
}

using NormGradients = std::tuple<at::Tensor, at::Tensor, std::optional<at::Tensor>>;
inline std::optional<NormGradients> layer_norm_backward(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& mean, const at::Tensor& rstd,
                                                        bool with_bias) {
    if (not_for_a_kernel({&dy, &x, &weight, &mean, &rstd})) return std::nullopt;
    LayerNormArgs a{};
    norm_rows(a, x, weight);
    TORCH_CHECK(dy.device() == x.device() && dy.scalar_type() == x.scalar_type() && dy.sizes() == x.sizes() && (dy.size(1) == 1 || dy.stride(1) == 1),
                "dy must be like x, with contiguous rows");
    for (const at::Tensor* t : {&mean, &rstd})
        TORCH_CHECK(t->device() == x.device() && t->scalar_type() == at::kFloat && t->is_contiguous() && t->dim() == 1 && t->size(0) == x.size(0),
                    "mean and rstd must be contiguous fp32 [rows] on the device of x");
    const c10::cuda::CUDAGuard guard(x.device());
    at::Tensor dx = at::empty({x.size(0), x.size(1)}, x.options());
    // (a storage each: they become the gradients of parameters, which are kept, saved and freed one by one)
    at::Tensor dw = at::empty({x.size(1)}, weight.options());
    std::optional<at::Tensor> db;
    if (with_bias) {
        db = at::empty({x.size(1)}, weight.options());
        a.db = db->data_ptr();
    }
    a.dy = dy.data_ptr();
    a.lddy = dy.stride(0);
    const NormShape shape = ep::layer_norm_backward_shape(a, device_sms());
    at::Tensor partial = at::empty({shape.ctas, with_bias ? 2 : 1, x.size(1)}, mean.options());
    a.mean = mean.data_ptr<float>();
    a.rstd = rstd.data_ptr<float>();
    a.dx = dx.data_ptr();
    a.dw = dw.data_ptr();
    a.partial = partial.data_ptr<float>();
    cuda_check(ep::launch_layer_norm_backward(a, shape, at::cuda::getCurrentCUDAStream()), "layer norm gradient launch");
    return NormGradients(dx, dw, db);
}

// Stack of matrices [count, rows, cols], bf16 or fp32, rows or columns contiguous -> bf16 [count, rows, cols]
inline at::Tensor orthogonalize(const at::Tensor& x, int64_t steps, double a, double b, double c, double eps, const std::optional<at::Tensor>& out, int64_t num_sms,
                                at::Tensor error, ElasticBufferCore* report_to) {
    TORCH_CHECK(x.is_cuda() && x.dim() == 3 && is_bf16_or_f32(x), "matrices must be bf16 or fp32 [count, rows, cols] on a GPU");
    TORCH_CHECK(steps >= 1, "at least one step");
    const int64_t count = x.size(0), R = x.size(1), C = x.size(2);
    TORCH_CHECK(count <= 65535 && R < (1ll << 20) && C < (1ll << 20), "at most 65535 matrices of fewer than 2^20 rows and columns");
    const bool by_rows = C == 1 ? R == 1 || x.stride(1) != 1 : x.stride(2) == 1;
    TORCH_CHECK(by_rows || R == 1 || x.stride(1) == 1, "rows or columns must be contiguous");
    const c10::cuda::CUDAGuard guard(x.device());
    at::Tensor res = out.has_value() ? *out : at::empty({count, R, C}, x.options().dtype(at::kBFloat16));
    TORCH_CHECK(res.device() == x.device() && res.scalar_type() == at::kBFloat16 && res.is_contiguous() && res.sizes() == x.sizes(),
                "out must be contiguous bf16 of the matrices' shape");
    if (res.numel() == 0) return res;
    TORCH_CHECK(reinterpret_cast<uintptr_t>(res.data_ptr()) % 16 == 0, "out must start on 16 bytes");
    NsArgs g{};
    const bool tall = R > C;
    g.in = x.data_ptr();
    g.in_bf16 = x.scalar_type() == at::kBFloat16;
    g.in_stride_matrix = x.stride(0);
    g.in_stride_line = by_rows ? x.stride(1) : x.stride(2);
    g.in_lines = by_rows ? R : C;
    g.in_line = static_cast<int>(by_rows ? C : R);
    g.flip = by_rows ? tall : !tall;
    g.out = res.data_ptr();
    g.out_transposed = tall;
    g.count = static_cast<int>(count);
    g.rows = static_cast<int>(std::min(R, C));
    g.cols = static_cast<int>(std::max(R, C));
    g.steps = static_cast<int>(std::min<int64_t>(steps, 1 << 30));
    g.a = static_cast<float>(a);
    g.b = static_cast<float>(b);
    g.c = static_cast<float>(c);
    TORCH_CHECK(ep::newton_schulz_fits(g), "singular values may grow beyond what the 16-bit operands of the products hold with these coefficients and steps");
    g.eps = static_cast<float>(eps);
    g.report.error = error.data_ptr<int>();
    if (report_to != nullptr) {
        report_to->check_status();
        const RankCtx ctx = report_to->ctx();
        g.report.status = ctx.status;
        g.report.status_rank = ctx.rank;
        g.report.timeout_ns = ctx.timeout_ns;
    }
    const int sms = num_sms > 0 ? static_cast<int>(std::min<int64_t>(num_sms, device_sms())) : device_sms();
    const NsWorkspace w = ep::newton_schulz_workspace(g, sms);
    at::Tensor workspace = at::empty({w.bytes}, x.options().dtype(at::kByte));
    cuda_check(ep::launch_newton_schulz(g, w, workspace.data_ptr<uint8_t>(), sms, at::cuda::getCurrentCUDAStream()), "orthogonalisation launch");
    return res;
}

}  // namespace ep_host
