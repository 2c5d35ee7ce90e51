// Tensor front end of the attention half of a layer: argument checks, result tensors, launches on the current stream.
#pragma once
#include <cmath>

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

// Scores are multiplied by scale log2 e in 32 bits: with zero there, those that are hidden (-inf) would be no numbers
inline void check_scale(double scale) {
    const float s = static_cast<float>(scale);
    TORCH_CHECK(s > 0 && std::isnormal(s) && std::isfinite(s * 1.5f), "scale must be positive, and neither too small nor too large for 32 bits");
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
    check_scale(scale);
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
                    q.size(0) * q.size(1) < (1ll << 34) && (q.size(0) / 128 + 1) * (q.size(1) / k.size(1)) < (1ll << 31), "too much work for one launch");
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
    a.num_sms = device_sms();
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
    cuda_check(ep::launch_attention(in.a, at::cuda::getCurrentCUDAStream()), "attention launch");
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
    TORCH_CHECK((q.size(0) / 128 + k.size(0) / 128 + 2 * static_cast<int64_t>(in.a.num_seqs)) * q.size(1) < (1ll << 31), "too much work for one launch");
    at::Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(k.sizes(), k.options());
    if (q.numel() == 0 || k.numel() == 0 || in.a.num_seqs == 0) return std::make_tuple(dq.zero_(), dk.zero_(), dv.zero_());
    const at::Tensor d16 = heads_of(d_o), o16 = heads_of(o);
    at::Tensor delta = at::empty(lse.sizes(), lse.options());
    in.a.d_o = view_of(d16);
    in.a.o_in = view_of(o16);
    in.a.lse_in = lse.data_ptr<float>();
    in.a.d_lse = d_lse.has_value() ? d_lse->data_ptr<float>() : nullptr;
    in.a.delta = delta.data_ptr<float>();
    in.a.splits = ep::attention_backward_splits(in.a);
    at::Tensor parts;
    if (in.a.splits > 1) {
        parts = at::empty({in.a.splits, 2, k.numel()}, lse.options());
        in.a.parts = parts.data_ptr<float>();
    }
    in.a.dq = dq.data_ptr();
    in.a.dk = dk.data_ptr();
    in.a.dv = dv.data_ptr();
    report_through(in.a.report, error, report_to);
    cuda_check(ep::launch_attention_backward(in.a, at::cuda::getCurrentCUDAStream()), "attention gradient launch");
    return std::make_tuple(dq, dk, dv);
}

// A caller's tensor has been written: who keeps it for a gradient hears of it, as of any operation in place
inline void note_written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// What paged caches [pages, page_size, kv_heads, dim] have to be
inline void check_caches(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& like, at::ScalarType type) {
    for (const at::Tensor* t : {&k_cache, &v_cache})
        TORCH_CHECK(t->device() == like.device() && t->scalar_type() == type && t->dim() == 4, "caches must be [pages, page_size, kv_heads, dim], of the type and on the device of the heads");
    TORCH_CHECK(k_cache.sizes() == v_cache.sizes() && k_cache.strides() == v_cache.strides(), "k_cache and v_cache must have one shape and one layout");
    TORCH_CHECK(k_cache.size(1) >= 1 && k_cache.size(1) < (1 << 30) && k_cache.size(0) < (1ll << 31), "between 1 and 2^30 places per page, fewer than 2^31 pages");
    TORCH_CHECK(k_cache.size(3) == 1 || k_cache.stride(3) == 1, "channels of the caches must be contiguous");
    const int64_t per16 = 16 / k_cache.element_size();
    for (int i = 0; i < 3; ++i) TORCH_CHECK(k_cache.stride(i) % per16 == 0, "heads of the caches must start on 16 bytes");
    for (const at::Tensor* t : {&k_cache, &v_cache}) TORCH_CHECK(reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0, "heads of the caches must start on 16 bytes");
}

inline at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& page_table, const at::Tensor& lengths, double scale,
                                  const std::optional<at::Tensor>& out) {
    TORCH_CHECK(q.is_cuda() && q.dim() == 3 && q.scalar_type() == at::kBFloat16, "q must be bf16 [sequences, heads, dim] on a GPU");
    const c10::cuda::CUDAGuard guard(q.device());
    check_caches(k_cache, v_cache, q, at::kBFloat16);
    const int64_t B = q.size(0), H = q.size(1), D = q.size(2), Hk = k_cache.size(2);
    TORCH_CHECK(D >= 8 && D <= 128 && D % 8 == 0 && k_cache.size(3) == D, "heads must have 8 to 128 channels, a multiple of 8, in q and the caches alike");
    TORCH_CHECK(H >= 1 && H < (1 << 16) && Hk >= 1 && H % Hk == 0, "the heads of q must be a multiple of those of the caches");
    TORCH_CHECK(B <= EP_MAX_PAGED_SEQS, "at most ", EP_MAX_PAGED_SEQS, " sequences");
    TORCH_CHECK(page_table.device() == q.device() && page_table.scalar_type() == at::kInt && page_table.dim() == 2 && page_table.size(0) == B &&
                    (page_table.size(1) <= 1 || page_table.stride(1) == 1) && page_table.size(1) < (1ll << 31),
                "page_table must be int32 [sequences, pages] with contiguous rows on the device of q");
    TORCH_CHECK(lengths.device() == q.device() && lengths.scalar_type() == at::kInt && lengths.dim() == 1 && lengths.size(0) == B && lengths.is_contiguous(),
                "lengths must be contiguous int32 [sequences] on the device of q");
    TORCH_CHECK(page_table.size(1) * k_cache.size(1) < (1ll << 31) - 65536 && B * (page_table.size(1) * k_cache.size(1) / 16 + 1) < (1ll << 31), "too many places in page_table");
    check_scale(scale);
    at::Tensor o = out.has_value() ? *out : at::empty(q.sizes(), q.options());
    TORCH_CHECK(o.device() == q.device() && o.scalar_type() == at::kBFloat16 && o.is_contiguous() && o.sizes() == q.sizes() && reinterpret_cast<uintptr_t>(o.data_ptr()) % 16 == 0,
                "out must be contiguous bf16 of q's shape, on 16 bytes");
    if (B == 0) return o;
    const at::Tensor q16 = heads_of(q);
    PagedAttentionArgs a{};
    a.q = view_of(q16);
    // (caches without pages have no address: nothing is read, and pointers are stepped from one that is there)
    a.k_cache = k_cache.numel() != 0 ? k_cache.data_ptr() : q16.data_ptr();
    a.v_cache = k_cache.numel() != 0 ? v_cache.data_ptr() : q16.data_ptr();
    a.stride_page = k_cache.stride(0);
    a.stride_slot = k_cache.stride(1);
    a.stride_head = k_cache.stride(2);
    a.num_pages = k_cache.size(0);
    a.page_size = static_cast<int>(k_cache.size(1));
    a.page_table = page_table.data_ptr<int>();
    a.table_pitch = page_table.stride(0);
    a.table_width = static_cast<int>(page_table.size(1));
    a.lengths = lengths.data_ptr<int>();
    a.num_seqs = static_cast<int>(B);
    a.heads = static_cast<int>(H);
    a.kv_heads = static_cast<int>(Hk);
    a.dim = static_cast<int>(D);
    a.scale = static_cast<float>(scale);
    a.o = o.data_ptr();
    at::Tensor parts;
    if (const int64_t bytes = ep::paged_attention_workspace(a, device_sms()); bytes > 0) {
        parts = at::empty({bytes}, q.options().dtype(at::kByte));
        a.parts = reinterpret_cast<float*>(parts.data_ptr());
    }
    cuda_check(ep::launch_paged_attention(a, device_sms(), at::cuda::getCurrentCUDAStream()), "paged attention launch");
    if (out.has_value()) note_written(o);
    return o;
}

// ------------------------------------------------------------------------------------------------ norm and rotation of heads
struct RotaryInputs {
    at::Tensor q, k, weight[2], table, positions;      // as the kernels read them
    RotaryArgs a{};
};
inline at::Tensor on16(const at::Tensor& t) { return t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone(at::MemoryFormat::Contiguous); }
inline RotaryInputs rotary_inputs(const at::Tensor& q, const at::Tensor& k, const at::Tensor& q_weight, const at::Tensor& k_weight, const at::Tensor& table, const at::Tensor& positions,
                                  double eps, bool interleaved) {
    for (const at::Tensor* t : {&q, &k})
        TORCH_CHECK(t->is_cuda() && t->device() == q.device() && t->dim() == 3 && is_bf16_or_f32(*t) && t->scalar_type() == q.scalar_type(),
                    "q and k must be bf16 or fp32 [tokens, heads, dim], of one type on one GPU");
    const int64_t T = q.size(0), D = q.size(2);
    TORCH_CHECK(k.size(0) == T && k.size(2) == D, "q and k must have the same tokens and channels");
    TORCH_CHECK(D >= 8 && D <= 256 && D % 8 == 0, "heads must have 8 to 256 channels, a multiple of 8");
    TORCH_CHECK(q.size(1) < (1 << 16) && k.size(1) < (1 << 16) && T < (1ll << 31) && T * (q.size(1) + 2 * k.size(1)) < (1ll << 31), "too many tokens or heads");
    for (const at::Tensor* t : {&q_weight, &k_weight})
        TORCH_CHECK(t->device() == q.device() && is_bf16_or_f32(*t) && t->scalar_type() == q_weight.scalar_type() && t->dim() == 1 && t->size(0) == D,
                    "weights must be bf16 or fp32 [dim], of one type, on the device of q");
    TORCH_CHECK(table.device() == q.device() && table.scalar_type() == at::kFloat && table.dim() == 2 && table.size(1) <= D && table.size(1) % 16 == 0,
                "table must be fp32 [positions, rotated channels], a multiple of 16 of at most dim, on the device of q");
    TORCH_CHECK(positions.device() == q.device() && positions.dim() == 1 && positions.size(0) == T && (positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt),
                "positions must be int64 or int32 [tokens] on the device of q");
    RotaryInputs in;
    in.q = heads_of(q);
    in.k = heads_of(k);
    in.weight[0] = on16(q_weight);
    in.weight[1] = on16(k_weight);
    in.table = on16(table);
    in.positions = positions.contiguous();
    RotaryArgs& a = in.a;
    a.x[0] = view_of(in.q);
    a.x[1] = view_of(in.k);
    a.heads[0] = static_cast<int>(q.size(1));
    a.heads[1] = static_cast<int>(k.size(1));
    for (int i = 0; i < 2; ++i) a.weight[i] = in.weight[i].data_ptr();
    a.tokens = static_cast<int>(T);
    a.dim = static_cast<int>(D);
    a.rotary = static_cast<int>(table.size(1));
    a.x_bf16 = q.scalar_type() == at::kBFloat16;
    a.param_bf16 = q_weight.scalar_type() == at::kBFloat16;
    a.interleaved = interleaved;
    a.table = in.table.data_ptr<float>();
    a.num_positions = table.size(0);
    a.positions = in.positions.data_ptr();
    a.positions_64 = in.positions.scalar_type() == at::kLong;
    a.eps = static_cast<float>(eps);
    return in;
}
// (nothing where a kernel is not to run, as of the norm)
inline std::optional<std::tuple<at::Tensor, at::Tensor>> qk_norm_rope(const at::Tensor& q, const at::Tensor& k, const at::Tensor& q_weight, const at::Tensor& k_weight,
                                                                      const at::Tensor& table, const at::Tensor& positions, double eps, bool interleaved) {
    if (not_for_a_kernel({&q, &k, &q_weight, &k_weight, &table}) || watched({&positions})) return std::nullopt;
    const c10::cuda::CUDAGuard guard(q.device());
    RotaryInputs in = rotary_inputs(q, k, q_weight, k_weight, table, positions, eps, interleaved);
    at::Tensor yq = at::empty(q.sizes(), q.options()), yk = at::empty(k.sizes(), k.options());
    if (q.numel() == 0 && k.numel() == 0) return std::make_tuple(yq, yk);
    in.a.out[0] = yq.data_ptr();
    in.a.out[1] = yk.data_ptr();
    cuda_check(ep::launch_rotary(in.a, device_sms(), at::cuda::getCurrentCUDAStream()), "rotation launch");
    return std::make_tuple(yq, yk);
}
inline std::optional<std::tuple<at::Tensor, std::optional<at::Tensor>>> qk_norm_rope_append(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& q_weight, const at::Tensor& k_weight,
                                                     const at::Tensor& table, const at::Tensor& positions, at::Tensor k_cache, at::Tensor v_cache, const at::Tensor& slots, double eps,
                                                     bool interleaved, bool keep_k) {
    if (not_for_a_kernel({&q, &k, &v, &q_weight, &k_weight, &table, &k_cache, &v_cache}) || watched({&positions, &slots})) return std::nullopt;
    const c10::cuda::CUDAGuard guard(q.device());
    RotaryInputs in = rotary_inputs(q, k, q_weight, k_weight, table, positions, eps, interleaved);
    TORCH_CHECK(v.device() == q.device() && v.scalar_type() == q.scalar_type() && v.sizes() == k.sizes(), "v must be like k");
    check_caches(k_cache, v_cache, q, q.scalar_type());
    TORCH_CHECK(k_cache.size(2) == k.size(1) && k_cache.size(3) == k.size(2), "the caches must have the heads and channels of k");
    for (int i = 0; i < 3; ++i) TORCH_CHECK(k_cache.size(i) <= 1 || k_cache.stride(i) > 0, "places and heads of the caches must not share memory");
    TORCH_CHECK(slots.device() == q.device() && slots.dim() == 1 && slots.size(0) == q.size(0) && (slots.scalar_type() == at::kLong || slots.scalar_type() == at::kInt),
                "slots must be int64 or int32 [tokens] on the device of q");
    at::Tensor yq = at::empty(q.sizes(), q.options());
    std::optional<at::Tensor> yk;
    if (keep_k) yk = at::empty(k.sizes(), k.options());
    if (q.numel() == 0 && k.numel() == 0) return std::make_tuple(yq, yk);
    const at::Tensor v16 = heads_of(v), s = slots.contiguous();
    RotaryArgs& a = in.a;
    a.out[0] = yq.data_ptr();
    if (keep_k) a.out[1] = yk->data_ptr();
    a.append = 1;
    a.v = view_of(v16);
    a.k_cache = k_cache.data_ptr();
    a.v_cache = v_cache.data_ptr();
    a.stride_page = k_cache.stride(0);
    a.stride_slot = k_cache.stride(1);
    a.stride_head = k_cache.stride(2);
    a.num_slots = k_cache.size(0) * k_cache.size(1);
    a.page_size = static_cast<int>(k_cache.size(1));
    a.slots = s.data_ptr();
    a.slots_64 = s.scalar_type() == at::kLong;
    cuda_check(ep::launch_rotary(a, device_sms(), at::cuda::getCurrentCUDAStream()), "rotation launch");
    note_written(k_cache);
    note_written(v_cache);
    return std::make_tuple(yq, yk);
}
using RotaryGradients = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>;
inline std::optional<RotaryGradients> qk_norm_rope_backward(const at::Tensor& dq, const at::Tensor& dk, const at::Tensor& q, const at::Tensor& k, const at::Tensor& q_weight,
                                                            const at::Tensor& k_weight, const at::Tensor& table, const at::Tensor& positions, double eps, bool interleaved) {
    if (not_for_a_kernel({&dq, &dk, &q, &k, &q_weight, &k_weight, &table}) || watched({&positions})) return std::nullopt;
    const c10::cuda::CUDAGuard guard(q.device());
    RotaryInputs in = rotary_inputs(q, k, q_weight, k_weight, table, positions, eps, interleaved);
    TORCH_CHECK(dq.device() == q.device() && dq.scalar_type() == q.scalar_type() && dq.sizes() == q.sizes() && dk.device() == q.device() && dk.scalar_type() == q.scalar_type() &&
                    dk.sizes() == k.sizes(), "gradients must be like q and k");
    at::Tensor dx = at::empty(q.sizes(), q.options()), dy = at::empty(k.sizes(), k.options());
    at::Tensor dqw = at::empty(q_weight.sizes(), q_weight.options()), dkw = at::empty(k_weight.sizes(), k_weight.options());
    if (q.numel() == 0 && k.numel() == 0) return RotaryGradients(dx, dy, dqw.zero_(), dkw.zero_());
    const at::Tensor dq16 = heads_of(dq), dk16 = heads_of(dk);
    RotaryArgs& a = in.a;
    a.dy[0] = view_of(dq16);
    a.dy[1] = view_of(dk16);
    a.out[0] = dx.data_ptr();
    a.out[1] = dy.data_ptr();
    a.dw[0] = dqw.data_ptr();
    a.dw[1] = dkw.data_ptr();
    a.ctas = ep::rotary_backward_ctas(a, device_sms());
    at::Tensor partial = at::empty({a.ctas, 2, a.dim}, table.options());
    a.partial = partial.data_ptr<float>();
    cuda_check(ep::launch_rotary_backward(a, at::cuda::getCurrentCUDAStream()), "rotation gradient launch");
    return RotaryGradients(dx, dy, dqw, dkw);
}

}  // namespace ep_host
