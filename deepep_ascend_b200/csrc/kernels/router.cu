// Routing of tokens to experts: scores, choice of the top-k experts (within the best groups), weights, tokens per expert; and the
// gradient of the weights with respect to the gate's logits.
//
//     p      = sigmoid(l), or exp(l - max l) / sum exp(l - max l)          (32 bits; the sum is a tree, see below)
//     choice = p + bias            nobody chooses an expert whose logit is -inf or whose choice is NaN or -inf
//     groups: the sum of a group's one or two best choices; the experts of the best groups stay
//     chosen = the num_topk best choices, equal ones by index;  w = scale * p (/ sum of the chosen p)
//
// The sum of the exponentials is a tree: the experts, padded with zeros to a power of two, are halved and the upper half is added to the lower one.
// That order is part of the definition: scores that differ in their last bit would choose another expert where two are as good.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "division.cuh"

namespace ep {

namespace {

constexpr float kNone = -__builtin_inff();

template <bool kBf16>
__device__ __forceinline__ float load_logit(const void* row, int e) {
    return kBf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[e]) : reinterpret_cast<const float*>(row)[e];
}

template <class T>
__device__ __forceinline__ T logit_of(float v) {
    if constexpr (sizeof(T) == 2) return __float2bfloat16_rn(v);
    else return v;
}

__device__ __forceinline__ float sigmoid(float l) { return __frcp_rn(1.f + expf(-l)); }

// (where reciprocal and quotient of division.cuh may be taken for the general ones)
constexpr float kLowLogit = -80.f;                               // 1 + exp(80) < 2^118
constexpr float kLowShare = 7.9e-31f;                            // over 2^-100

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
    float r;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float min8_nan(const float (&v)[8]) {
    const float a = min3_nan(v[0], v[1], v[2]), b = min3_nan(v[3], v[4], v[5]);
    return min3_nan(a, b, min3_nan(v[6], v[7], v[7]));
}
__device__ __forceinline__ float max_nan(float a, float b) {      // a NaN wins, as everything computed with it is one
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// over the eight lanes of a token
template <class F>
__device__ __forceinline__ float over8(float v, F f) {
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float sum8(float v) {
    return over8(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Eight neighbouring logits; those past the end are -inf.  kWide: rows start on 16 bytes and end with a whole eight.
template <bool kBf16, bool kWide>
__device__ __forceinline__ void load8(const void* row, int first, int experts, float (&v)[8]) {
    if constexpr (kWide && kBf16) {
        const uint4 q = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(row) + first);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else if constexpr (kWide) {
        const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(row) + first);
        const float4 b = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(row) + first + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = first + i < experts ? load_logit<kBf16>(row, first + i) : kNone;
    }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void fetch8(const float* p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

// Shared memory of a warp, which works on up to four tokens at a time: the choices of each (for a softmax an odd number of eights apart, so
// that the four tokens' lanes, eight each, meet different banks); the best and second best of each eight; the groups' scores.
constexpr int kTokens = 4;
struct RouteLayout {
    int eights, pitch, best, group, warp;       // eights of a token; floats from token to token; offsets in floats of the warp's arrays; floats of a warp
};
__host__ __device__ inline RouteLayout route_layout(int experts, int groups, bool softmax) {
    RouteLayout l;
    l.eights = (experts + 7) / 8;
    l.pitch = (softmax ? l.eights | 1 : l.eights) * 8;
    l.best = kTokens * l.pitch;
    l.group = l.best + kTokens * 2 * ((l.eights + 3) / 4 * 4);
    l.warp = l.group + (groups > 1 ? kTokens * 32 : 0);
    return l;
}
// leaf(0) + ... + leaf(kCount - 1), the upper half added to the lower one until one is left
template <int kCount, int kFirst = 0, int kStep = 1, class F>
__device__ __forceinline__ float sum_by_halves(const F& leaf) {
    if constexpr (kStep >= kCount) return leaf(kFirst);
    else return sum_by_halves<kCount, kFirst, kStep * 2>(leaf) + sum_by_halves<kCount, kFirst + kStep, kStep * 2>(leaf);
}

// A warp takes `tokens` (1 or 4) at a time.  Scores: a lane has eight neighbouring experts of one token.  Choice: eight lanes per token, each with kSegs eights
// of which it knows the largest choice; a chosen expert is found, taken out, and the new largest of its eight made by the token's eight lanes together, so that the
// shuffles of a step serve four tokens.  Bound by instruction issue (1720 per warp and four tokens, 70 % of the issue slots; DRAM 18 %): about a third are the
// exact exponentials and reciprocals, a quarter the steps of the choice.
// 65536 x 256 fp32, 8 of 256 in 4 of 8 groups: 42 us, 1.8 TB/s (softmax 55); one token per warp, with a maximum over the warp for every expert, took 139, steps that
// branch 48.  Requesting the next tokens' logits into L2 ahead gained nothing (43).
// CTAs per SM: as many as leave the registers (64, or 80 for more than 256 experts) for what a lane holds: 32768 x 512 with 64 took 81 us instead of 72.
template <int kSegs, bool kBf16, bool kWide, bool kSoftmax>
__global__ void __launch_bounds__(256, kSegs > 4 ? 3 : 4) route_kernel(const RouterArgs a, const int tokens) {
    extern __shared__ __align__(16) float route_smem[];
    const RouteLayout l = route_layout(a.num_experts, a.num_groups, kSoftmax);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, E = a.num_experts, K = a.num_topk, S = l.eights, G = a.num_groups;
    float* mine = route_smem + warp * l.warp;
    float *choice = mine, *best = mine + l.best, *group_score = mine + l.group;
    const int P = kSoftmax ? l.pitch : S * 8;
    auto place = [&](int u, int t, int seg) { return kSoftmax ? t * P + seg * 8 : u * 8; };      // of an eight
    const int best_pitch = (S + 3) / 4 * 4;
    float* second = best + kTokens * best_pitch;
    float* s_bias = route_smem + warps * l.warp;                              // [S * 8]
    int* s_count = reinterpret_cast<int*>(s_bias + S * 8);                    // [E]
    for (int e = threadIdx.x; e < E; e += blockDim.x) s_count[e] = 0;
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    int odd = 0;
    for (int e = threadIdx.x; e < S * 8; e += blockDim.x) {
        s_bias[e] = a.bias != nullptr && e < E ? a.bias[e] : 0.f;
        odd |= !(fabsf(s_bias[e]) < -kNone);
    }
    // eights past the last one of a token, which the lanes below look at, hold nobody
    for (int i = lane; i < 2 * kTokens * best_pitch; i += 32) best[i] = kNone;
    const bool odd_bias = __syncthreads_or(odd) != 0;
    const int size = E / G;                            // experts of a group
    const bool whole = G > 1 && size % 8 == 0;         // groups of whole eights
    const int t8 = lane >> 3, q = lane & 7;            // token and place of the lane where eight lanes have a token
    int seg_group[kSegs];
#pragma unroll
    for (int i = 0; i < kSegs; ++i) seg_group[i] = whole ? min(q * kSegs + i, S - 1) * 8 / size : 0;
    const float inverse_g = 1.f / G;
    uint32_t token_of = 0;                             // of this lane's eights lane, lane + 32, ... of four tokens: two bits each
#pragma unroll
    for (int i = 0; i < kSegs; ++i) token_of |= static_cast<uint32_t>(min((lane + 32 * i) / S, kTokens - 1)) << (2 * i);
    // largest and second largest choice of an eight
    auto tops = [&](const float (&c)[8], int t, int seg) {
        float hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) hi[i] = fmaxf(c[i], c[i + 4]), lo[i] = fminf(c[i], c[i + 4]);
#pragma unroll
        for (int h = 2; h > 0; h /= 2)
#pragma unroll
            for (int i = 0; i < h; ++i) {
                lo[i] = max3(lo[i], lo[i + h], fminf(hi[i], hi[i + h]));
                hi[i] = fmaxf(hi[i], hi[i + h]);
            }
        best[t * best_pitch + seg] = hi[0];
        second[t * best_pitch + seg] = lo[0];
    };
    // A choice that is no number, or whose logit is -inf, is nobody's.  Looked at one by one, with the general reciprocal or quotient, only in an eight
    // that has others than ordinary numbers, or where the bias has.
    auto settled = [](float logit, float c) { return c > kNone && logit > kNone ? c : kNone; };

    const int64_t step = static_cast<int64_t>(gridDim.x) * warps * tokens;
    for (int64_t t0 = (static_cast<int64_t>(blockIdx.x) * warps + warp) * tokens; t0 < a.num_tokens; t0 += step) {
        const int n = static_cast<int>(min(static_cast<int64_t>(tokens), a.num_tokens - t0)), units = n * S;
        const uint8_t* rows = reinterpret_cast<const uint8_t*>(a.logits) + t0 * a.ld * (kBf16 ? 2 : 4);
        const int64_t pitch = a.ld * (kBf16 ? 2 : 4);
        float top = 0.f, total = 1.f;                  // of the token of this lane's eight
        if constexpr (kSoftmax) {
            // logits, and the largest of each eight
            for (uint32_t w = token_of, u = lane; u < static_cast<uint32_t>(units); u += 32, w >>= 2) {
                const int t = w & 3, seg = u - t * S;
                float v[8];
                load8<kBf16, kWide>(rows + t * pitch, seg * 8, E, v);
                store8(choice + place(u, t, seg), v);
                best[t * best_pitch + seg] = max_nan(max_nan(max_nan(v[0], v[1]), max_nan(v[2], v[3])), max_nan(max_nan(v[4], v[5]), max_nan(v[6], v[7])));
            }
            __syncwarp();
            top = kNone;
            if (t8 < n)
                for (int s = q; s < S; s += 8) top = max_nan(top, best[t8 * best_pitch + s]);
            top = over8(top, max_nan);
            // exp(l - max) of the lane's experts q, q + 8, ..., and their sum.  (With zeros up to 64 kSegs experts the tree has the same sum.)
            total = 0.f;
            if (t8 < n) {
                float* e = choice + t8 * P + q;
                total = sum_by_halves<8 * kSegs>([&](int s) {
                    if (s >= S) return 0.f;
                    return e[s * 8] = expf(e[s * 8] - top);
                });
            }
            total = sum8(total);
            __syncwarp();
            for (uint32_t w = token_of, u0 = 0; u0 < static_cast<uint32_t>(units); u0 += 32, w >>= 2) {
                const int u = u0 + lane, t = w & 3, seg = u - t * S;
                const float sum = __shfl_sync(0xffffffffu, total, t * 8);
                if (u < units) {
                    float c[8], b[8];
                    fetch8(choice + place(u, t, seg), c);
                    fetch8(s_bias + seg * 8, b);
                    if (!odd_bias && min8_nan(c) >= kLowShare) {       // (none of a logit that is -inf)
                        const float inverse = reciprocal(sum);
#pragma unroll
                        for (int i = 0; i < 8; ++i) c[i] = quotient(c[i], sum, inverse) + b[i];
                    } else {
                        float logit[8];
                        load8<kBf16, kWide>(rows + t * pitch, seg * 8, E, logit);
#pragma unroll
                        for (int i = 0; i < 8; ++i) c[i] = settled(logit[i], __fdiv_rn(c[i], sum) + b[i]);
                    }
                    store8(choice + place(u, t, seg), c);
                    tops(c, t, seg);
                }
            }
        } else {
            for (uint32_t w = token_of, u = lane; u < static_cast<uint32_t>(units); u += 32, w >>= 2) {
                const int t = w & 3, seg = u - t * S;
                float logit[8], c[8], b[8];
                load8<kBf16, kWide>(rows + t * pitch, seg * 8, E, logit);
                fetch8(s_bias + seg * 8, b);
                if (!odd_bias && min8_nan(logit) >= kLowLogit) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) c[i] = reciprocal(1.f + expf(-logit[i])) + b[i];
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) c[i] = settled(logit[i], sigmoid(logit[i]) + b[i]);
                }
                store8(choice + place(u, t, seg), c);
                tops(c, t, seg);
            }
        }
        __syncwarp();
        uint32_t kept = 0xffffffffu;                   // groups of token t8 that stay
        if (G > 1) {
            // scores of the groups: their two best
            for (int u = lane; u < n * G; u += 32) {
                const int t = static_cast<int>((u + 0.5f) * inverse_g), g = u - t * G;
                float v1 = kNone, v2 = kNone;
                if (whole) {
                    for (int s = g * (size / 8); s < (g + 1) * (size / 8); ++s) {
                        const float b1 = best[t * best_pitch + s], b2 = second[t * best_pitch + s];
                        v2 = fmaxf(fminf(v1, b1), fmaxf(v2, b2));
                        v1 = fmaxf(v1, b1);
                    }
                } else {
                    const float* c = choice + t * P + g * size;
                    for (int i = 0; i < size; ++i) {
                        v2 = fmaxf(v2, fminf(v1, c[i]));
                        v1 = fmaxf(v1, c[i]);
                    }
                }
                group_score[t * 32 + g] = a.group_top == 2 && v2 > kNone ? v1 + v2 : v1;
            }
            __syncwarp();
            // the groups that fewer than num_topk_groups others beat, equal ones by index; eight lanes per token
            kept = 0;
            if (t8 < n)
                for (int g = q; g < G; g += 8) {
                    const float score = group_score[t8 * 32 + g];
                    int better = 0;
                    for (int h = 0; h < G; ++h) {
                        const float other = group_score[t8 * 32 + h];
                        better += other > score || (other == score && h < g);
                    }
                    if (better < a.num_topk_groups) kept |= 1u << g;
                }
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) kept |= __shfl_xor_sync(0xffffffffu, kept, o);
            if (!whole) {
                // groups that end within an eight: their experts leave one by one
                for (uint32_t w = token_of, u0 = 0; u0 < static_cast<uint32_t>(units); u0 += 32, w >>= 2) {
                    const int u = u0 + lane, t = w & 3, seg = u - t * S;
                    const uint32_t stay = __shfl_sync(0xffffffffu, kept, t * 8);
                    if (u < units) {
                        float c[8];
                        fetch8(choice + place(u, t, seg), c);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (((stay >> min((seg * 8 + i) / size, 31)) & 1u) == 0) c[i] = kNone;
                        store8(choice + place(u, t, seg), c);
                        tops(c, t, seg);
                    }
                }
                kept = 0xffffffffu;
                __syncwarp();
            }
        }
        // the largest choice of each of this lane's eights
        float m[kSegs];
        const bool routed = t8 < n && (a.token_mask == nullptr || a.token_mask[t0 + t8] != 0);
#pragma unroll
        for (int i = 0; i < kSegs; ++i) {
            const int seg = q * kSegs + i;
            m[i] = routed && seg < S && ((kept >> seg_group[i]) & 1u) != 0 ? best[t8 * best_pitch + seg] : kNone;
        }
        int chosen[2] = {-1, -1};                      // experts q and q + 8 of token t8
        float* c8 = choice + (t8 < n ? t8 : 0) * P + q;
        const uint32_t ours = 0xffu << (t8 * 8);       // this token's lanes
        const auto larger = [](float x, float y) { return fmaxf(x, y); };
#pragma unroll 1
        for (int k = 0; k < K; ++k) {
            float largest = m[0];
#pragma unroll
            for (int i = 1; i < kSegs; ++i) largest = fmaxf(largest, m[i]);
            const float wanted = over8(largest, larger);
            // the first eight that has it, and there the first expert
            const int owner = __ffs(__ballot_sync(0xffffffffu, largest == wanted) & ours) - 1;
            int at = 0;
#pragma unroll
            for (int i = kSegs - 1; i > 0; --i)
                if (m[i] == wanted) at = i;
            if (m[0] == wanted) at = 0;
            const int seg = __shfl_sync(0xffffffffu, q * kSegs + at, owner);
            // (selects, not branches: a step has little else to do than to wait for its shuffles)
            const bool some = wanted > kNone;
            float* place_c = c8 + seg * 8;
            const float seen = *place_c;
            const int hit = __ffs(__ballot_sync(0xffffffffu, some && seen == wanted) & ours) - 1;
            const bool taken = lane == hit;
            if (taken) *place_c = kNone;
            const float next = over8(some && !taken ? seen : kNone, larger);
            const bool owns = lane == owner;
#pragma unroll
            for (int i = 0; i < kSegs; ++i) m[i] = owns && i == at ? next : m[i];          // (nobody left: -inf takes its own place)
            const int id = some ? seg * 8 + (hit & 7) : -1;
            chosen[0] = q == k ? id : chosen[0];
            chosen[1] = q + 8 == k ? id : chosen[1];
        }
        // weights: the lane's first expert, and its second one where a token has more than eight
        const uint8_t* row = rows + (t8 < n ? t8 : 0) * pitch;
        const bool two = K > 8;
        float logit[2] = {kNone, kNone}, p[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if ((i == 0 || two) && chosen[i] >= 0) logit[i] = load_logit<kBf16>(row, chosen[i]);
        if constexpr (kSoftmax) {
            // renormalised weights are taken relative to the largest chosen logit: also right where p itself would vanish
            if (a.renormalize) top = over8(max_nan(logit[0], logit[1]), max_nan), total = 1.f;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if ((i == 0 || two) && chosen[i] >= 0) {
                p[i] = kSoftmax ? __fdiv_rn(expf(logit[i] - top), total) : sigmoid(logit[i]);
                atomicAdd(&s_count[chosen[i]], 1);
            }
        const float sum = a.renormalize ? sum8(p[0] + p[1]) : 1.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int k = q + i * 8;
            if ((i == 0 || two) && t8 < n && k < K) {
                const int64_t out = (t0 + t8) * K + k;
                if (a.idx_is_64) reinterpret_cast<int64_t*>(a.topk_idx)[out] = chosen[i];
                else reinterpret_cast<int32_t*>(a.topk_idx)[out] = chosen[i];
                if (a.renormalize) p[i] = sum > 0.f ? __fdiv_rn(p[i], sum) : 0.f;
                a.topk_weights[out] = p[i] * a.scale;
            }
        }
        __syncwarp();
    }
    __syncthreads();
    // the only CTA of a small batch has all counts; otherwise they are added to a cleared array
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
        if (gridDim.x == 1) a.count[e] = s_count[e];
        else if (s_count[e] != 0) atomicAdd(&a.count[e], s_count[e]);
    }
}

// ------------------------------------------------------------------------------------------------ gradient
// d loss / d logits of a row.  sigmoid: dp p (1 - p) at the chosen experts; softmax with renormalised weights: the other experts' scores
// cancel, w (dw - sum dw w) at the chosen ones; softmax as it is: p (dp - sum dp p) for every expert.

__device__ __forceinline__ int chosen_expert(const RouterArgs& a, int64_t at) {
    const int64_t e = a.idx_is_64 ? reinterpret_cast<const int64_t*>(a.topk_idx)[at] : reinterpret_cast<const int32_t*>(a.topk_idx)[at];
    return e >= 0 && e < a.num_experts ? static_cast<int>(e) : -1;
}

// Gradients that only chosen experts have.  A warp takes kRows tokens at a time, eight lanes for each of four; their rows, zero but for the chosen experts,
// lie in shared memory and leave as one bulk copy (kRows rows start and end on 16 bytes for any number of experts), two sets of rows in turn.  What is
// left to do per row is to write and clear its few values.  65536 x 256 fp32, 8 chosen: 20 us, 3.8 TB/s; rows put together in registers took 42.
template <bool kBf16>
__global__ void __launch_bounds__(256) route_backward_kernel(const RouterArgs a) {
    using T = std::conditional_t<kBf16, __nv_bfloat16, float>;
    constexpr int kRows = kBf16 ? 8 : 4, kSets = 2;
    extern __shared__ __align__(16) uint8_t route_rows[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, E = a.num_experts, K = a.num_topk;
    const int t8 = lane >> 3, q = lane & 7;
    const int set_bytes = kRows * E * static_cast<int>(sizeof(T));
    uint8_t* mine = route_rows + warp * kSets * set_bytes;
    for (int i = lane; i < kSets * set_bytes / 16; i += 32) reinterpret_cast<uint4*>(mine)[i] = make_uint4(0, 0, 0, 0);
    __syncwarp();
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    constexpr int kParts = kRows / 4;
    int held[kSets][kParts][2];                        // where this lane's values lie
#pragma unroll
    for (int s = 0; s < kSets; ++s)
#pragma unroll
        for (int p = 0; p < kParts; ++p) held[s][p][0] = held[s][p][1] = -1;
    const int64_t step = static_cast<int64_t>(gridDim.x) * warps * kRows;
    int64_t t0 = (static_cast<int64_t>(blockIdx.x) * warps + warp) * kRows;
    // Ids, weights' gradients and then logits wait for one another: ids come two batches ahead, logits one
    struct Batch {
        int expert[kParts][2];
        float dw[kParts][2], logit[kParts][2];
    };
    const bool two = K > 8;
    auto request_ids = [&](Batch& b, int64_t first) {
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int64_t t = first + p * 4 + t8;
                b.expert[p][i] = -1;
                b.dw[p][i] = 0.f;
                if ((i == 0 || two) && t < a.num_tokens && q + i * 8 < K) {
                    const int64_t at = t * K + q + i * 8;
                    b.expert[p][i] = chosen_expert(a, at);
                    b.dw[p][i] = a.d_weights[at];
                }
            }
    };
    auto request_logits = [&](Batch& b, int64_t first) {
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                b.logit[p][i] = b.expert[p][i] >= 0 ? load_logit<kBf16>(reinterpret_cast<const uint8_t*>(a.logits) + (first + p * 4 + t8) * a.ld * sizeof(T), b.expert[p][i]) : kNone;
    };
    Batch batch[3];
    request_ids(batch[0], t0);
    request_ids(batch[1], t0 + step);
    request_logits(batch[0], t0);
    int s = 0;
    for (; t0 < a.num_tokens; t0 += step, s ^= 1) {
        request_logits(batch[1], t0 + step);
        request_ids(batch[2], t0 + 2 * step);
        const Batch& b = batch[0];
        const int n = static_cast<int>(min(static_cast<int64_t>(kRows), a.num_tokens - t0));
        T* rows = reinterpret_cast<T*>(mine + s * set_bytes);
        float d[kParts][2];
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
            float w[2] = {0.f, 0.f}, dw[2], slope[2] = {1.f, 1.f};
            // relative to the largest chosen logit: w = p / sum p needs no other
            const float top = a.softmax ? over8(max_nan(b.logit[p][0], b.logit[p][1]), max_nan) : 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                dw[i] = b.expert[p][i] >= 0 ? b.dw[p][i] * a.scale : 0.f;
                if ((i == 0 || two) && b.expert[p][i] >= 0) {
                    w[i] = a.softmax ? expf(b.logit[p][i] - top) : sigmoid(b.logit[p][i]);
                    if (!a.softmax) slope[i] = sigmoid(-b.logit[p][i]);
                }
            }
            float along = 0.f;
            if (a.renormalize) {
                const float sum = sum8(w[0] + w[1]);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (i == 0 || two) w[i] = sum > 0.f ? __fdiv_rn(w[i], sum) : 0.f;
                along = sum8(dw[0] * w[0] + dw[1] * w[1]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) d[p][i] = w[i] * (dw[i] - along) * slope[i];
        }
        // the copy that last read this set has ended; its values go, the new ones come
        if (lane == 0) ptx::bulk_wait_read<kSets - 1>();
        __syncwarp();
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int old = s == 0 ? held[0][p][i] : held[1][p][i];
                if (old >= 0) rows[old] = logit_of<T>(0.f);
            }
        __syncwarp();
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = b.expert[p][i] >= 0 ? (p * 4 + t8) * E + b.expert[p][i] : -1;
                if (s == 0) held[0][p][i] = at;
                else held[1][p][i] = at;
                if (at >= 0) rows[at] = logit_of<T>(d[p][i]);
            }
        T* out = reinterpret_cast<T*>(a.d_logits) + t0 * E;
        const int bytes = n * E * static_cast<int>(sizeof(T));
        if (bytes % 16 == 0) {
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) ptx::bulk_store(out, rows, bytes);
        } else {
            __syncwarp();
            for (int i = lane; i < n * E; i += 32) out[i] = rows[i];
        }
        if (lane == 0) ptx::bulk_commit();
        batch[0] = batch[1];
        batch[1] = batch[2];
    }
    if (lane == 0) ptx::bulk_wait_read<0>();
}

// Softmax weights as they are: every expert's logit has a gradient.  One warp per token; lane i has the experts i, i + 32, ...
template <int kVals, bool kBf16>
__global__ void __launch_bounds__(256) route_backward_all_kernel(const RouterArgs a) {
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5, E = a.num_experts, K = a.num_topk;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * warps + (threadIdx.x >> 5); t < a.num_tokens; t += static_cast<int64_t>(gridDim.x) * warps) {
        const uint8_t* row = reinterpret_cast<const uint8_t*>(a.logits) + t * a.ld * (kBf16 ? 2 : 4);
        const int expert = lane < K ? chosen_expert(a, t * K + lane) : -1;
        float out[kVals];
#pragma unroll
        for (int j = 0; j < kVals; ++j) out[j] = 0.f;
        if (__ballot_sync(0xffffffffu, expert >= 0) != 0) {
            const float dw = expert >= 0 ? a.d_weights[t * K + lane] * a.scale : 0.f;
            float top = kNone, sum = 0.f;
#pragma unroll
            for (int j = 0; j < kVals; ++j) {
                out[j] = j * 32 + lane < E ? load_logit<kBf16>(row, j * 32 + lane) : kNone;
                top = max_nan(top, out[j]);
            }
            top = warp_max_nan(top);
#pragma unroll
            for (int j = 0; j < kVals; ++j) sum += out[j] = expf(out[j] - top);
            const float inverse = 1.f / warp_sum(sum);
            const float d = expert >= 0 ? expf(load_logit<kBf16>(row, expert) - top) * inverse * dw : 0.f;
            const float along = -warp_sum(d) * inverse;
#pragma unroll
            for (int j = 0; j < kVals; ++j) out[j] *= along;
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

using RouteKernel = void (*)(RouterArgs, int);
template <bool kBf16, bool kWide, bool kSoftmax>
RouteKernel route_kernel_of(int experts) {
    if (experts <= 64) return route_kernel<1, kBf16, kWide, kSoftmax>;
    if (experts <= 128) return route_kernel<2, kBf16, kWide, kSoftmax>;
    if (experts <= 256) return route_kernel<4, kBf16, kWide, kSoftmax>;
    if (experts <= 512) return route_kernel<8, kBf16, kWide, kSoftmax>;
    return route_kernel<16, kBf16, kWide, kSoftmax>;
}
template <bool kBf16>
RouteKernel route_kernel_of(int experts, bool wide, bool softmax) {
    if (wide) return softmax ? route_kernel_of<kBf16, true, true>(experts) : route_kernel_of<kBf16, true, false>(experts);
    return softmax ? route_kernel_of<kBf16, false, true>(experts) : route_kernel_of<kBf16, false, false>(experts);
}
using RouterKernel = void (*)(RouterArgs);
template <bool kBf16>
RouterKernel backward_all_of(int experts) {
    if (experts <= 32) return route_backward_all_kernel<1, kBf16>;
    if (experts <= 64) return route_backward_all_kernel<2, kBf16>;
    if (experts <= 128) return route_backward_all_kernel<4, kBf16>;
    if (experts <= 256) return route_backward_all_kernel<8, kBf16>;
    if (experts <= 512) return route_backward_all_kernel<16, kBf16>;
    return route_backward_all_kernel<32, kBf16>;
}

bool bad_router_args(const RouterArgs& a) {
    return a.num_experts < 1 || a.num_experts > EP_MAX_EXPERTS || a.num_topk < 1 || a.num_topk > EP_MAX_TOPK || a.num_tokens < 0 || a.ld < a.num_experts;
}

// CTAs of a launch, and leave for its shared memory.  Nothing is asked for small launches that need neither: it is a tenth of what they take.
cudaError_t grid_of(const void* fn, int threads, int smem, int64_t ctas, int num_sms, int& grid) {
    int per_sm = 1;
    const cudaError_t err = ctas <= num_sms && smem <= 48 * 1024 ? cudaSuccess : allow_shared_memory(fn, threads, smem, &per_sm);
    grid = static_cast<int>(std::min<int64_t>(ctas, static_cast<int64_t>(num_sms) * per_sm));
    return err;
}
// warps of a CTA: eight, or as many as have room
int warps_of(int bytes_per_warp, int bytes) { return std::max(1, std::min(8, (200 * 1024 - bytes) / bytes_per_warp)); }

}  // namespace

cudaError_t launch_route(const RouterArgs& args, int num_sms, cudaStream_t stream) {
    RouterArgs a = args;
    if (bad_router_args(a) || a.num_groups < 1 || a.num_groups > 32 || a.num_experts % a.num_groups != 0 || a.num_topk_groups < 1 || a.num_topk_groups > a.num_groups ||
        a.group_top < 1 || a.group_top > 2)
        return cudaErrorInvalidValue;
    if (a.num_tokens == 0) return cudaMemsetAsync(a.count, 0, sizeof(int32_t) * a.num_experts, stream);
    const int size = a.logits_bf16 ? 2 : 4;
    const bool wide = a.num_experts % 8 == 0 && a.ld * size % 16 == 0 && reinterpret_cast<uintptr_t>(a.logits) % 16 == 0;
    const RouteKernel kernel = a.logits_bf16 ? route_kernel_of<true>(a.num_experts, wide, a.softmax != 0) : route_kernel_of<false>(a.num_experts, wide, a.softmax != 0);
    const void* fn = reinterpret_cast<const void*>(kernel);
    const RouteLayout l = route_layout(a.num_experts, a.num_groups, a.softmax != 0);
    const int shared = 4 * (l.eights * 8 + a.num_experts);
    // four tokens per warp where every SM gets some warps of them
    int tokens = a.num_tokens >= 4 * 4 * num_sms ? kTokens : 1;
    int warps = warps_of(4 * l.warp, shared);
    if (a.num_tokens <= warps * tokens) warps = std::max(1, (a.num_tokens + tokens - 1) / tokens);
    const int smem = warps * 4 * l.warp + shared;
    const int64_t per_cta = static_cast<int64_t>(warps) * tokens, ctas = (a.num_tokens + per_cta - 1) / per_cta;
    int grid = 1;
    cudaError_t err = grid_of(fn, warps * 32, smem, ctas, num_sms, grid);
    if (err != cudaSuccess) return err;
    if (grid > 1) err = cudaMemsetAsync(a.count, 0, sizeof(int32_t) * a.num_experts, stream);
    if (err != cudaSuccess) return err;
    void* params[] = {&a, &tokens};
    return launch_dependent(fn, dim3(grid), dim3(warps * 32), params, smem, stream);
}

cudaError_t launch_route_backward(const RouterArgs& args, int num_sms, cudaStream_t stream) {
    RouterArgs a = args;
    if (bad_router_args(a)) return cudaErrorInvalidValue;
    if (a.num_tokens == 0) return cudaSuccess;
    void* params[] = {&a};
    if (a.softmax && !a.renormalize) {
        const RouterKernel kernel = a.logits_bf16 ? backward_all_of<true>(a.num_experts) : backward_all_of<false>(a.num_experts);
        const int64_t ctas = (a.num_tokens + 7) / 8;
        return launch_dependent(reinterpret_cast<const void*>(kernel), dim3(static_cast<unsigned>(std::min<int64_t>(ctas, 8ll * num_sms))), dim3(256), params, 0, stream);
    }
    if (reinterpret_cast<uintptr_t>(a.d_logits) % 16 != 0) return cudaErrorInvalidValue;
    const RouterKernel kernel = a.logits_bf16 ? route_backward_kernel<true> : route_backward_kernel<false>;
    const void* fn = reinterpret_cast<const void*>(kernel);
    const int rows = a.logits_bf16 ? 8 : 4, per_warp = 2 * rows * a.num_experts * (a.logits_bf16 ? 2 : 4), warps = warps_of(per_warp, 0), smem = warps * per_warp;
    const int64_t ctas = (a.num_tokens + warps * rows - 1) / (warps * rows);
    int grid = 1;
    const cudaError_t err = grid_of(fn, warps * 32, smem, ctas, num_sms, grid);
    if (err != cudaSuccess) return err;
    return launch_dependent(fn, dim3(grid), dim3(warps * 32), params, smem, stream);
}

}  // namespace ep
