// Routing of tokens to experts: scores, choice of the top-k experts (within the best groups), weights, tokens per expert; and the
// gradient of the weights with respect to the gate's logits.
//
//     p      = sigmoid(l), or exp(l - max l) / sum exp(l - max l)          (32 bits; the sum is a tree, see below)
//     choice = p + bias            nobody chooses an expert whose logit is -inf or whose choice is NaN or -inf
//     groups: the sum of a group's one or two best choices; the experts of the best groups stay
//     chosen = the num_topk best choices, equal ones by index;  w = scale * p (/ sum of the chosen p)
//
// One warp per token.  Lane i of a warp holds the experts i, i + 32, ...: every load of the warp is contiguous, and the sum of the
// exponentials "upper half added to lower half" has its first levels within a lane and the others across lanes.  That order is part of the
// definition: scores that differ in their last bit would choose another expert where two are as good.
#include <math_constants.h>

#include <algorithm>

#include "common.cuh"

namespace ep {

namespace {

constexpr int kRouterWarps = 8;

template <bool kBf16>
__device__ __forceinline__ float load_logit(const void* row, int e) {
    return kBf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[e]) : reinterpret_cast<const float*>(row)[e];
}

__device__ __forceinline__ float sigmoid(float l) { return __frcp_rn(1.f + expf(-l)); }

__device__ __forceinline__ float warp_max_nan(float v) {      // a NaN wins, as everything computed with it is one
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(v), "f"(w));
    }
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// floats as integers of the same order (no NaN, no -0)
__device__ __forceinline__ int order_key(float v) {
    const int b = __float_as_int(v);
    return b ^ ((b >> 31) & 0x7fffffff);
}

// the row's softmax: maximum and sum of exp(l - max); v[j] becomes exp(l - max)
template <int kVals>
__device__ __forceinline__ void softmax_row(float (&v)[kVals], int lane, int experts, float& top, float& total) {
    top = -CUDART_INF_F;
#pragma unroll
    for (int j = 0; j < kVals; ++j)
        if (j * 32 + lane < experts) asm("max.NaN.f32 %0, %1, %2;" : "=f"(top) : "f"(top), "f"(v[j]));
    top = warp_max_nan(top);
    float sum[kVals];
#pragma unroll
    for (int j = 0; j < kVals; ++j) sum[j] = v[j] = j * 32 + lane < experts ? expf(v[j] - top) : 0.f;
#pragma unroll
    for (int h = kVals / 2; h > 0; h >>= 1)
#pragma unroll
        for (int j = 0; j < h; ++j) sum[j] += sum[j + h];
    total = warp_sum(sum[0]);
}

template <int kVals, bool kBf16>
__global__ void __launch_bounds__(kRouterWarps * 32) route_kernel(const RouterArgs a) {
    extern __shared__ uint8_t router_smem[];
    int* s_count = reinterpret_cast<int*>(router_smem);                                 // [experts]
    float* s_choice = reinterpret_cast<float*>(s_count + a.num_experts);                // [warps][experts], with groups
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = a.num_experts, K = a.num_topk;
    for (int e = threadIdx.x; e < E; e += blockDim.x) s_count[e] = 0;
    __syncthreads();
    s_choice += warp * E;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * kRouterWarps + warp; t < a.num_tokens; t += static_cast<int64_t>(gridDim.x) * kRouterWarps) {
        int my_expert = -1;
        float my_p = 0.f;
        if (a.token_mask == nullptr || a.token_mask[t] != 0) {
            const uint8_t* row = reinterpret_cast<const uint8_t*>(a.logits) + t * a.ld * (kBf16 ? 2 : 4);
            float c[kVals];
            uint32_t off = 0;                   // bit j: expert j * 32 + lane cannot be chosen
#pragma unroll
            for (int j = 0; j < kVals; ++j) {
                const int e = j * 32 + lane;
                c[j] = e < E ? load_logit<kBf16>(row, e) : -CUDART_INF_F;
                if (c[j] == -CUDART_INF_F) off |= 1u << j;
            }
            float top = 0.f, total = 1.f;
            if (a.softmax) {
                softmax_row<kVals>(c, lane, E, top, total);
#pragma unroll
                for (int j = 0; j < kVals; ++j) c[j] = __fdiv_rn(c[j], total);
            } else {
#pragma unroll
                for (int j = 0; j < kVals; ++j) c[j] = sigmoid(c[j]);
            }
#pragma unroll
            for (int j = 0; j < kVals; ++j) {
                const int e = j * 32 + lane;
                if (a.bias != nullptr && e < E) c[j] += a.bias[e];
                if (((off >> j) & 1u) != 0 || isnan(c[j])) c[j] = -CUDART_INF_F;
            }
            if (a.num_groups > 1) {
                const int G = a.num_groups, size = E / G;
#pragma unroll
                for (int j = 0; j < kVals; ++j)
                    if (j * 32 + lane < E) s_choice[j * 32 + lane] = c[j];
                __syncwarp();
                float v1 = -CUDART_INF_F, v2 = -CUDART_INF_F;
                if (lane < G)
                    for (int i = 0; i < size; ++i) {
                        const float v = s_choice[lane * size + i];
                        v2 = fmaxf(v2, fminf(v1, v));
                        v1 = fmaxf(v1, v);
                    }
                const float score = a.group_top == 2 && v2 != -CUDART_INF_F ? v1 + v2 : v1;
                int better = 0;
                for (int g = 0; g < G; ++g) {
                    const float other = __shfl_sync(0xffffffffu, score, g);
                    better += other > score || (other == score && g < lane);
                }
                const uint32_t keep = __ballot_sync(0xffffffffu, lane < G && better < a.num_topk_groups);
#pragma unroll
                for (int j = 0; j < kVals; ++j) {
                    const int e = j * 32 + lane;
                    if (e < E && ((keep >> (e / size)) & 1u) == 0) c[j] = -CUDART_INF_F;
                }
                __syncwarp();
            }
            for (int k = 0; k < K; ++k) {
                float best = -CUDART_INF_F;
                int at = E;
#pragma unroll
                for (int j = 0; j < kVals; ++j)
                    if (c[j] > best) best = c[j], at = j * 32 + lane;
                const int key = order_key(best), top_key = __reduce_max_sync(0xffffffffu, key);
                const int e = __reduce_min_sync(0xffffffffu, key == top_key ? at : E);
                if (e >= E) break;              // nobody is left
                if (lane == k) my_expert = e;
#pragma unroll
                for (int j = 0; j < kVals; ++j)
                    if (j * 32 + lane == e) c[j] = -CUDART_INF_F;
            }
            const float l = my_expert >= 0 ? load_logit<kBf16>(row, my_expert) : -CUDART_INF_F;
            // renormalised softmax weights are taken relative to the largest chosen logit: also right where p itself would vanish
            if (a.softmax && a.renormalize) top = warp_max_nan(l), total = 1.f;
            if (my_expert >= 0) {
                my_p = a.softmax ? __fdiv_rn(expf(l - top), total) : sigmoid(l);
                atomicAdd(&s_count[my_expert], 1);
            }
        }
        float w = my_p;
        if (a.renormalize) {
            const float sum = warp_sum(my_p);
            w = sum > 0.f ? __fdiv_rn(my_p, sum) : 0.f;
        }
        if (lane < K) {
            if (a.idx_is_64) reinterpret_cast<int64_t*>(a.topk_idx)[t * K + lane] = my_expert;
            else reinterpret_cast<int32_t*>(a.topk_idx)[t * K + lane] = my_expert;
            a.topk_weights[t * K + lane] = w * a.scale;
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += blockDim.x)
        if (s_count[e] != 0) atomicAdd(&a.count[e], s_count[e]);
}

// d loss / d logits of a row.  sigmoid: dp p (1 - p) at the chosen experts; softmax with renormalised weights: the other experts' scores
// cancel, w (dw - sum dw w) at the chosen ones; softmax as it is: p (dp - sum dp p) for every expert.
template <int kVals, bool kBf16>
__global__ void __launch_bounds__(kRouterWarps * 32) route_backward_kernel(const RouterArgs a) {
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = a.num_experts, K = a.num_topk;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * kRouterWarps + warp; t < a.num_tokens; t += static_cast<int64_t>(gridDim.x) * kRouterWarps) {
        const uint8_t* row = reinterpret_cast<const uint8_t*>(a.logits) + t * a.ld * (kBf16 ? 2 : 4);
        int expert = -1;
        float dw = 0.f;
        if (lane < K) {
            const int64_t e = a.idx_is_64 ? reinterpret_cast<const int64_t*>(a.topk_idx)[t * K + lane] : reinterpret_cast<const int32_t*>(a.topk_idx)[t * K + lane];
            if (e >= 0 && e < E) {
                expert = static_cast<int>(e);
                dw = a.d_weights[t * K + lane] * a.scale;
            }
        }
        float out[kVals];
#pragma unroll
        for (int j = 0; j < kVals; ++j) out[j] = 0.f;
        if (__ballot_sync(0xffffffffu, expert >= 0) != 0) {
            const float l = expert >= 0 ? load_logit<kBf16>(row, expert) : 0.f;
            float d;
            if (!a.softmax || a.renormalize) {
                float p = 0.f, slope = 1.f;
                if (a.softmax) {
                    // relative to the largest chosen logit: w = p / sum p needs no other
                    const float top = warp_max_nan(expert >= 0 ? l : -CUDART_INF_F);
                    p = expert >= 0 ? expf(l - top) : 0.f;
                } else if (expert >= 0) {
                    p = sigmoid(l);
                    slope = sigmoid(-l);
                }
                if (a.renormalize) {
                    const float sum = warp_sum(p), w = sum > 0.f ? __fdiv_rn(p, sum) : 0.f;
                    d = w * (dw - warp_sum(dw * w)) * slope;
                } else {
                    d = dw * p * slope;
                }
            } else {
                float c[kVals], top, total;
#pragma unroll
                for (int j = 0; j < kVals; ++j) c[j] = j * 32 + lane < E ? load_logit<kBf16>(row, j * 32 + lane) : 0.f;
                softmax_row<kVals>(c, lane, E, top, total);
                const float p = expert >= 0 ? __fdiv_rn(expf(l - top), total) : 0.f;
                const float along = warp_sum(dw * p);
#pragma unroll
                for (int j = 0; j < kVals; ++j) out[j] = -along * __fdiv_rn(c[j], total);
                d = p * dw;
            }
            for (int k = 0; k < K; ++k) {
                const int e = __shfl_sync(0xffffffffu, expert, k);
                const float v = __shfl_sync(0xffffffffu, d, k);
#pragma unroll
                for (int j = 0; j < kVals; ++j)
                    if (j * 32 + lane == e) out[j] += v;
            }
        }
#pragma unroll
        for (int j = 0; j < kVals; ++j) {
            const int e = j * 32 + lane;
            if (e < E) {
                if (kBf16) reinterpret_cast<__nv_bfloat16*>(a.d_logits)[t * E + e] = __float2bfloat16_rn(out[j]);
                else reinterpret_cast<float*>(a.d_logits)[t * E + e] = out[j];
            }
        }
    }
}

using RouterKernel = void (*)(RouterArgs);
template <bool kBackward, bool kBf16>
RouterKernel router_kernel(int experts) {
    if (experts <= 32) return kBackward ? route_backward_kernel<1, kBf16> : route_kernel<1, kBf16>;
    if (experts <= 64) return kBackward ? route_backward_kernel<2, kBf16> : route_kernel<2, kBf16>;
    if (experts <= 128) return kBackward ? route_backward_kernel<4, kBf16> : route_kernel<4, kBf16>;
    if (experts <= 256) return kBackward ? route_backward_kernel<8, kBf16> : route_kernel<8, kBf16>;
    if (experts <= 512) return kBackward ? route_backward_kernel<16, kBf16> : route_kernel<16, kBf16>;
    return kBackward ? route_backward_kernel<32, kBf16> : route_kernel<32, kBf16>;
}

bool bad_router_args(const RouterArgs& a) {
    return a.num_experts < 1 || a.num_experts > EP_MAX_EXPERTS || a.num_topk < 1 || a.num_topk > EP_MAX_TOPK || a.num_tokens < 0 || a.ld < a.num_experts;
}

}  // namespace

cudaError_t launch_route(const RouterArgs& a, int num_sms, cudaStream_t stream) {
    if (bad_router_args(a) || a.num_groups < 1 || a.num_groups > 32 || a.num_experts % a.num_groups != 0 || a.num_topk_groups < 1 || a.num_topk_groups > a.num_groups ||
        a.group_top < 1 || a.group_top > 2)
        return cudaErrorInvalidValue;
    cudaError_t err = cudaMemsetAsync(a.count, 0, sizeof(int32_t) * a.num_experts, stream);
    if (err != cudaSuccess || a.num_tokens == 0) return err;
    const RouterKernel fn = a.logits_bf16 ? router_kernel<false, true>(a.num_experts) : router_kernel<false, false>(a.num_experts);
    const size_t smem = sizeof(int) * a.num_experts * (a.num_groups > 1 ? 1 + kRouterWarps : 1);
    const int64_t ctas = (a.num_tokens + kRouterWarps - 1) / kRouterWarps;
    void* params[] = {const_cast<RouterArgs*>(&a)};
    return launch_dependent(reinterpret_cast<const void*>(fn), dim3(static_cast<unsigned>(std::min<int64_t>(ctas, 8ll * num_sms))), dim3(kRouterWarps * 32), params, smem, stream);
}

cudaError_t launch_route_backward(const RouterArgs& a, int num_sms, cudaStream_t stream) {
    if (bad_router_args(a)) return cudaErrorInvalidValue;
    if (a.num_tokens == 0) return cudaSuccess;
    const RouterKernel fn = a.logits_bf16 ? router_kernel<true, true>(a.num_experts) : router_kernel<true, false>(a.num_experts);
    const int64_t ctas = (a.num_tokens + kRouterWarps - 1) / kRouterWarps;
    void* params[] = {const_cast<RouterArgs*>(&a)};
    return launch_dependent(reinterpret_cast<const void*>(fn), dim3(static_cast<unsigned>(std::min<int64_t>(ctas, 8ll * num_sms))), dim3(kRouterWarps * 32), params, 0, stream);
}

}  // namespace ep
