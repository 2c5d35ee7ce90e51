// Tensor front end of the attention half of a layer: argument checks, result tensors, launches on the current stream.
#pragma once
#include "block_ops.hpp"

namespace ep_host {

// Heads [tokens, heads, dim] whose channels are contiguous and whose rows start on 16 bytes, as bulk copies and 16-byte accesses need them: `t` itself, or a copy
inline at::Tensor heads_of(const at::Tensor& t) {
    bool fits = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && (t.size(2) == 1 || t.stride(2) == 1);
    const int64_t per16 = 16 / t.element_size();
    for (int i = 0; i < 2; ++i) fits = fits && (t.size(i) <= 1 || (t.stride(i) > 0 && t.stride(i) % per16 == 0));
    if (fits || t.numel() == 0) return t;
    at::Tensor copy = at::empty(t.sizes(), t.options());
    copy.copy_(t);
    return copy;
}
inline HeadsView view_of(const at::Tensor& t) { return HeadsView{t.data_ptr(), t.stride(0), t.stride(1)}; }

inline void report_through(NsReport& report, at::Tensor& error, ElasticBufferCore* report_to) {
    report.error = error.data_ptr<int>();
    if (report_to != nullptr) {
        report_to->check_status();
        const RankCtx ctx = report_to->ctx();
        report.status = ctx.status;
        report.status_rank = ctx.rank;
        report.timeout_ns = ctx.timeout_ns;
    }
}

struct PackedInputs {
    at::Tensor q, k, v;                // as the kernels read them
    AttentionArgs a{};
};
inline PackedInputs packed_inputs(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const std::optional<at::Tensor>& cu_q, const std::optional<at::Tensor>& cu_k,
                                  bool causal, double scale) {
    for (const at::Tensor* t : {&q, &k, &v})
        TORCH_CHECK(t->is_cuda() && t->device() == q.device() && t->dim() == 3 && t->scalar_type() == at::kBFloat16, "q, k and v must be bf16 [tokens, heads, dim] on one GPU");
    TORCH_CHECK(k.sizes() == v.sizes() && q.size(2) == k.size(2), "k and v must have one shape, and the channels of q");
    TORCH_CHECK(q.size(2) >= 8 && q.size(2) <= 128 && q.size(2) % 8 == 0, "heads must have 8 to 128 channels, a multiple of 8");
    TORCH_CHECK(k.size(1) >= 1 && q.size(1) >= 1 && q.size(1) % k.size(1) == 0, "the heads of q must be a multiple of those of k");
    TORCH_CHECK(q.size(0) < (1ll << 30) && k.size(0) < (1ll << 30) && q.size(1) < (1 << 16), "too many tokens or heads");
    TORCH_CHECK(std::isfinite(scale) && scale > 0, "scale must be positive");
    TORCH_CHECK(cu_q.has_value() == cu_k.has_value(), "cu_seqlens of queries and keys go together");
    PackedInputs in;
    AttentionArgs& a = in.a;
    a.num_seqs = 1;
    if (cu_q.has_value()) {
        for (const at::Tensor* t : {&*cu_q, &*cu_k})
            TORCH_CHECK(t->device() == q.device() && t->scalar_type() == at::kInt && t->dim() == 1 && t->is_contiguous() && t->size(0) >= 1 && t->sizes() == cu_q->sizes(),
                        "cu_seqlens must be contiguous int32 [sequences + 1] on the device of q, for queries and keys alike");
        a.num_seqs = static_cast<int>(cu_q->size(0) - 1);
        a.cu_q = cu_q->data_ptr<int>();
        a.cu_k = cu_k->data_ptr<int>();
    }
    TORCH_CHECK((q.size(0) / 128 + a.num_seqs) * q.size(1) < (1ll << 31) && (k.size(0) / 128 + a.num_seqs) * q.size(1) < (1ll << 31) &&
                    q.size(0) * q.size(1) < (1ll << 34), "too much work for one launch");
    in.q = heads_of(q);
    in.k = heads_of(k);
    in.v = heads_of(v);
    a.q = view_of(in.q);
    a.k = view_of(in.k);
    a.v = view_of(in.v);
    a.tq = static_cast<int>(q.size(0));
    a.tk = static_cast<int>(k.size(0));
    a.heads = static_cast<int>(q.size(1));
    a.kv_heads = static_cast<int>(k.size(1));
    a.dim = static_cast<int>(q.size(2));
    a.causal = causal;
    a.scale = static_cast<float>(scale);
    return in;
}

// (nothing where a kernel is not to run, as of the norm)
inline std::optional<std::tuple<at::Tensor, at::Tensor>> attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const std::optional<at::Tensor>& cu_q,
                                                                   const std::optional<at::Tensor>& cu_k, bool causal, double scale, at::Tensor error,
                                                                   ElasticBufferCore* report_to) {
    const c10::cuda::CUDAGuard guard(q.device());
    PackedInputs in = packed_inputs(q, k, v, cu_q, cu_k, causal, scale);
    at::Tensor o = at::empty(q.sizes(), q.options()), lse = at::empty({q.size(1), q.size(0)}, q.options().dtype(at::kFloat));
    if (q.size(0) == 0) return std::make_tuple(o, lse);
    if (k.size(0) == 0 || in.a.num_seqs == 0) return std::make_tuple(o.zero_(), lse.fill_(-std::numeric_limits<float>::infinity()));
    in.a.o = o.data_ptr();
    in.a.lse = lse.data_ptr<float>();
    report_through(in.a.report, error, report_to);
    cuda_check(ep::launch_attention(in.a, device_sms(), at::cuda::getCurrentCUDAStream()), "attention launch");
    return std::make_tuple(o, lse);
}

inline std::optional<std::tuple<at::Tensor, at::Tensor, at::Tensor>> attention_backward(const at::Tensor& d_o, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                                                        const at::Tensor& o, const at::Tensor& lse, const std::optional<at::Tensor>& d_lse,
                                                                                        const std::optional<at::Tensor>& cu_q, const std::optional<at::Tensor>& cu_k, bool causal,
                                                                                        double scale, at::Tensor error, ElasticBufferCore* report_to) {
    const c10::cuda::CUDAGuard guard(q.device());
    PackedInputs in = packed_inputs(q, k, v, cu_q, cu_k, causal, scale);
    for (const at::Tensor* t : {&d_o, &o})
        TORCH_CHECK(t->device() == q.device() && t->scalar_type() == at::kBFloat16 && t->sizes() == q.sizes(), "o and its gradient must be like q");
    TORCH_CHECK(lse.device() == q.device() && lse.scalar_type() == at::kFloat && lse.is_contiguous() && lse.dim() == 2 && lse.size(0) == q.size(1) && lse.size(1) == q.size(0),
                "lse must be contiguous fp32 [heads, tokens] on the device of q");
    if (d_lse.has_value())
        TORCH_CHECK(d_lse->device() == q.device() && d_lse->scalar_type() == at::kFloat && d_lse->is_contiguous() && d_lse->sizes() == lse.sizes(),
                    "the gradient of lse must be like lse, and contiguous");
    at::Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(k.sizes(), k.options());
    if (q.numel() == 0 || k.numel() == 0 || in.a.num_seqs == 0) return std::make_tuple(dq.zero_(), dk.zero_(), dv.zero_());
    const at::Tensor d16 = heads_of(d_o), o16 = heads_of(o);
    at::Tensor delta = at::empty(lse.sizes(), lse.options());
    in.a.d_o = view_of(d16);
    in.a.o_in = view_of(o16);
    in.a.lse_in = lse.data_ptr<float>();
    in.a.d_lse = d_lse.has_value() ? d_lse->data_ptr<float>() : nullptr;
    in.a.delta = delta.data_ptr<float>();
    in.a.dq = dq.data_ptr();
    in.a.dk = dk.data_ptr();
    in.a.dv = dv.data_ptr();
    report_through(in.a.report, error, report_to);
    cuda_check(ep::launch_attention_backward(in.a, device_sms(), at::cuda::getCurrentCUDAStream()), "attention gradient launch");
    return std::make_tuple(dq, dk, dv);
}

}  // namespace ep_host
