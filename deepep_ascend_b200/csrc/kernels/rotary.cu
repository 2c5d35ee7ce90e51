// RMS norm of every query and key head and rotation of its channels by the token's position, in one pass, and its gradient.  Per head x of D channels, with the weight w:
//
//     rstd = (mean x^2 + eps)^-1/2,   n = rstd x w,   (a, b) of a pair of channels -> (a cos - b sin, b cos + a sin)
//
// where the pairs are channels (i, i + R/2) of the first R channels, or, interleaved, (2 i, 2 i + 1).  Backwards: g = dy rotated back,
//
//     dw = sum over tokens and heads of g rstd x,     u = g w,     dx = rstd (u - rstd^2 x mean(u x))
//
// Bound by memory: every value is read once and written once.  A row of D channels lies on 8, 16 or 32 lanes of a warp, eight channels each; partners that are R/2 apart
// exchange their raw values (four registers of bf16 pairs, where normed ones would take eight) and norm them on both sides.
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace ep {

namespace {

using bf16 = __nv_bfloat16;
constexpr int kRotaryThreads = 256;

template <class T>
struct Eight {
    uint4 raw[sizeof(T) / 2];
};
template <class T>
__device__ __forceinline__ Eight<T> load8(const T* p) {
    Eight<T> e;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) e.raw[i] = reinterpret_cast<const uint4*>(p)[i];
    return e;
}
__device__ __forceinline__ void to_float(const Eight<bf16>& e, float (&f)[8]) {
    const uint32_t w[4] = {e.raw[0].x, e.raw[0].y, e.raw[0].z, e.raw[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void to_float(const Eight<float>& e, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        f[4 * i] = __uint_as_float(e.raw[i].x);
        f[4 * i + 1] = __uint_as_float(e.raw[i].y);
        f[4 * i + 2] = __uint_as_float(e.raw[i].z);
        f[4 * i + 3] = __uint_as_float(e.raw[i].w);
    }
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
    if constexpr (sizeof(T) == 2) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(f[2 * i + 1]), "f"(f[2 * i]));
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
}
// those of lane `from`
template <class T>
__device__ __forceinline__ Eight<T> exchange(const Eight<T>& e, int from) {
    Eight<T> r;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
        r.raw[i].x = __shfl_sync(0xffffffffu, e.raw[i].x, from);
        r.raw[i].y = __shfl_sync(0xffffffffu, e.raw[i].y, from);
        r.raw[i].z = __shfl_sync(0xffffffffu, e.raw[i].z, from);
        r.raw[i].w = __shfl_sync(0xffffffffu, e.raw[i].w, from);
    }
    return r;
}
__device__ __forceinline__ void load_weight(const void* w, int is_bf16, int c, float (&f)[8]) {
    if (is_bf16) to_float(load8(static_cast<const bf16*>(w) + c), f);
    else to_float(load8(static_cast<const float*>(w) + c), f);
}
__device__ __forceinline__ int64_t load_index(const void* p, int is_64, int64_t i) {
    return is_64 ? static_cast<const int64_t*>(p)[i] : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
}
template <int kLanes>
__device__ __forceinline__ float sum_row(float v) {
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// What a lane knows of its place in the rows
template <int kLanes, bool kInterleaved>
struct Place {
    static constexpr int kRows = 32 / kLanes;            // rows of a warp
    int sub, c, partner, angle;                          // row of the warp, first channel, lane of the partners, first angle
    bool on, turned, second;                             // lanes that hold channels, that hold rotated ones, whose are the second of their pairs
    __device__ __forceinline__ Place(int dim, int rotary) {
        const int lane = threadIdx.x & 31, in = lane % kLanes;
        sub = lane / kLanes;
        c = in * 8;
        on = c < dim;
        turned = c < rotary;
        second = !kInterleaved && c >= rotary / 2;
        partner = kInterleaved || !turned ? lane : lane + (second ? -rotary / 16 : rotary / 16);
        angle = kInterleaved ? c / 2 : (second ? c - rotary / 2 : c);
    }
};
// Cosines and sines of a lane's pairs; rows of zeros in front of the table, of no numbers behind it
template <bool kInterleaved>
struct Angles {
    static constexpr int kCount = kInterleaved ? 4 : 8;
    float cos[kCount], sin[kCount], keep;
    template <class P>
    __device__ __forceinline__ Angles(const RotaryArgs& a, const P& place, int64_t position) {
        keep = position < 0 ? 0.f : (position < a.num_positions ? 1.f : __int_as_float(0x7fc00000));
        const float* row = a.table + (position >= 0 && position < a.num_positions ? position : 0) * a.rotary + place.angle;
#pragma unroll
        for (int i = 0; i < kCount; i += 4) {
            const bool read = place.turned && a.num_positions > 0;
            const float4 u = read ? *reinterpret_cast<const float4*>(row + i) : make_float4(1.f, 1.f, 1.f, 1.f);
            const float4 v = read ? *reinterpret_cast<const float4*>(row + a.rotary / 2 + i) : make_float4(0.f, 0.f, 0.f, 0.f);
            cos[i] = u.x, cos[i + 1] = u.y, cos[i + 2] = u.z, cos[i + 3] = u.w;
            sin[i] = v.x, sin[i + 1] = v.y, sin[i + 2] = v.z, sin[i + 3] = v.w;
        }
    }
};

// Rows [kIters] of a warp: heads of one kind (queries, keys, values) of one token
template <class T, int kLanes, bool kInterleaved, int kIters>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ RotaryArgs a, int chunks_q, int chunks_k, int chunks) {
    using Lane = Place<kLanes, kInterleaved>;
    constexpr int kHeads = kIters * Lane::kRows;
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kRotaryThreads / 32) + (threadIdx.x >> 5);
    const int64_t token = unit / chunks;
    if (token >= a.tokens) return;
    int chunk = static_cast<int>(unit - token * chunks);
    const int kind = chunk < chunks_q ? 0 : (chunk < chunks_q + chunks_k ? 1 : 2);
    chunk -= kind == 0 ? 0 : (kind == 1 ? chunks_q : chunks_q + chunks_k);
    const Lane place(a.dim, a.rotary);
    const float inv_dim = 1.f / a.dim;
    const HeadsView& x = kind == 2 ? a.v : a.x[kind];
    const int heads = a.heads[kind == 0 ? 0 : 1], head0 = chunk * kHeads + place.sub;
    Eight<T> raw[kIters] = {};
#pragma unroll
    for (int i = 0; i < kIters; ++i)
        if (place.on && head0 + i * Lane::kRows < heads)
            raw[i] = load8(static_cast<const T*>(x.data) + token * x.stride_token + (head0 + i * Lane::kRows) * x.stride_head + place.c);
    T* out;
    int64_t pitch;
    bool write = place.on;
    if (kind == 0 || a.k_cache == nullptr) {
        out = static_cast<T*>(a.out[kind]) + token * heads * a.dim;
        pitch = a.dim;
    } else {
        const int64_t slot = load_index(a.slots, a.slots_64, token);
        write = write && slot >= 0 && slot < a.num_slots;
        const int64_t page = slot / a.page_size;
        out = static_cast<T*>(kind == 1 ? a.k_cache : a.v_cache) + page * a.stride_page + (slot - page * a.page_size) * a.stride_slot;
        pitch = a.stride_head;
    }
    if (kind == 2) {
#pragma unroll
        for (int i = 0; i < kIters; ++i)
            if (write && head0 + i * Lane::kRows < heads) {
                T* row = out + (head0 + i * Lane::kRows) * pitch + place.c;
#pragma unroll
                for (int j = 0; j < static_cast<int>(sizeof(T)) / 2; ++j) reinterpret_cast<uint4*>(row)[j] = raw[i].raw[j];
            }
        return;
    }
    const Angles<kInterleaved> turn(a, place, load_index(a.positions, a.positions_64, token));
    float w[8] = {}, w_partner[8] = {};
    if (place.on) load_weight(a.weight[kind], a.param_bf16, place.c, w);
    if (!kInterleaved && place.turned) load_weight(a.weight[kind], a.param_bf16, place.second ? place.c - a.rotary / 2 : place.c + a.rotary / 2, w_partner);
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
        float v[8], y[8], squares = 0.f;
        to_float(raw[i], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) squares = fmaf(v[j], v[j], squares);
        const float rstd = __frsqrt_rn(sum_row<kLanes>(squares) * inv_dim + a.eps);
        if constexpr (kInterleaved) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = v[2 * j] * rstd * w[2 * j], q = v[2 * j + 1] * rstd * w[2 * j + 1];
                y[2 * j] = p * turn.cos[j] - q * turn.sin[j];
                y[2 * j + 1] = q * turn.cos[j] + p * turn.sin[j];
            }
        } else {
            float u[8];
            to_float(exchange(raw[i], place.partner), u);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float p = v[j] * rstd * w[j], q = u[j] * rstd * w_partner[j];
                y[j] = p * turn.cos[j] + (place.second ? q : -q) * turn.sin[j];
            }
        }
        if (turn.keep != 1.f)
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = turn.keep;
        if (write && head0 + i * Lane::kRows < heads) store8(out + (head0 + i * Lane::kRows) * pitch + place.c, y);
    }
}

// Gradient: a warp takes chunks of heads, those of queries and then those of keys, and keeps its sums of the weight's gradient
template <class T, int kLanes, bool kInterleaved, int kIters>
__global__ void __launch_bounds__(kRotaryThreads) rotary_backward_kernel(const __grid_constant__ RotaryArgs a) {
    using Lane = Place<kLanes, kInterleaved>;
    constexpr int kHeads = kIters * Lane::kRows, kWarps = kRotaryThreads / 32;
    __shared__ float s_sum[kWarps][kLanes * 8];
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const Lane place(a.dim, a.rotary);
    const float inv_dim = 1.f / a.dim;
    const int warp = threadIdx.x >> 5;
#pragma unroll 1
    for (int kind = 0; kind < 2; ++kind) {
        const int heads = a.heads[kind], chunks = (heads + kHeads - 1) / kHeads;
        const int64_t units = static_cast<int64_t>(a.tokens) * chunks;
        float w[8] = {}, dw[8] = {};
        if (place.on) load_weight(a.weight[kind], a.param_bf16, place.c, w);
#pragma unroll 1
        for (int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + warp; unit < units; unit += static_cast<int64_t>(gridDim.x) * kWarps) {
            const int64_t token = unit / chunks;
            const int head0 = static_cast<int>(unit - token * chunks) * kHeads + place.sub;
            Eight<T> x[kIters] = {}, d[kIters] = {};
#pragma unroll
            for (int i = 0; i < kIters; ++i)
                if (place.on && head0 + i * Lane::kRows < heads) {
                    const int64_t head = head0 + i * Lane::kRows;
                    x[i] = load8(static_cast<const T*>(a.x[kind].data) + token * a.x[kind].stride_token + head * a.x[kind].stride_head + place.c);
                    d[i] = load8(static_cast<const T*>(a.dy[kind].data) + token * a.dy[kind].stride_token + head * a.dy[kind].stride_head + place.c);
                }
            const Angles<kInterleaved> turn(a, place, load_index(a.positions, a.positions_64, token));
#pragma unroll
            for (int i = 0; i < kIters; ++i) {
                float v[8], g[8], own[8];
                to_float(x[i], v);
                to_float(d[i], own);
                if constexpr (kInterleaved) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        g[2 * j] = own[2 * j] * turn.cos[j] + own[2 * j + 1] * turn.sin[j];
                        g[2 * j + 1] = own[2 * j + 1] * turn.cos[j] - own[2 * j] * turn.sin[j];
                    }
                } else {
                    float u[8];
                    to_float(exchange(d[i], place.partner), u);
#pragma unroll
                    for (int j = 0; j < 8; ++j) g[j] = own[j] * turn.cos[j] + (place.second ? -u[j] : u[j]) * turn.sin[j];
                }
                if (turn.keep != 1.f)
#pragma unroll
                    for (int j = 0; j < 8; ++j) g[j] = turn.keep;
                float squares = 0.f, along = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    squares = fmaf(v[j], v[j], squares);
                    along = fmaf(g[j] * w[j], v[j], along);
                }
                squares = sum_row<kLanes>(squares);
                along = sum_row<kLanes>(along);
                const float rstd = __frsqrt_rn(squares * inv_dim + a.eps), back = rstd * rstd * (along * inv_dim);
                float dx[8];
                if (head0 + i * Lane::kRows < heads) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        dx[j] = rstd * (g[j] * w[j] - v[j] * back);
                        dw[j] = turn.keep == 0.f ? dw[j] : fmaf(g[j] * rstd, v[j], dw[j]);
                    }
                    if (place.on) {
                        if (turn.keep == 0.f)
#pragma unroll
                            for (int j = 0; j < 8; ++j) dx[j] = 0.f;
                        store8(static_cast<T*>(a.out[kind]) + (token * heads + head0 + i * Lane::kRows) * a.dim + place.c, dx);
                    }
                }
            }
        }
        // rows of a warp, then warps
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int o = kLanes; o < 32; o <<= 1) dw[j] += __shfl_xor_sync(0xffffffffu, dw[j], o);
        __syncthreads();
        if (place.sub == 0)
#pragma unroll
            for (int j = 0; j < 8; ++j) s_sum[warp][place.c + j] = dw[j];
        __syncthreads();
        for (int c = threadIdx.x; c < a.dim; c += kRotaryThreads) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < kWarps; ++i) sum += s_sum[i][c];
            a.partial[(static_cast<int64_t>(blockIdx.x) * 2 + kind) * a.dim + c] = sum;
        }
    }
}

// The CTAs' sums of 32 channels: 32 warps take every 32nd CTA
__global__ void __launch_bounds__(1024) rotary_reduce_kernel(const __grid_constant__ RotaryArgs a) {
    __shared__ float s_sum[32][33];
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, at = blockIdx.x * 32 + lane;
    float sum = 0.f;
    if (at < 2 * a.dim)
#pragma unroll 8
        for (int i = warp; i < a.ctas; i += 32) sum += a.partial[static_cast<int64_t>(i) * 2 * a.dim + at];
    s_sum[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && at < 2 * a.dim) {
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) sum += s_sum[i][lane];
        const int kind = at >= a.dim, c = at - kind * a.dim;
        if (a.param_bf16) static_cast<bf16*>(a.dw[kind])[c] = __float2bfloat16_rn(sum);
        else static_cast<float*>(a.dw[kind])[c] = sum;
    }
}

constexpr int kForwardIters = 4, kBackwardIters = 2;
int lanes_of(int dim) { return dim <= 64 ? 8 : (dim <= 128 ? 16 : 32); }

template <class F>
cudaError_t with_shape(const RotaryArgs& a, F f) {
    auto types = [&](auto lanes, auto interleaved) { return a.x_bf16 ? f(bf16{}, lanes, interleaved) : f(float{}, lanes, interleaved); };
    auto pairs = [&](auto lanes) { return a.interleaved ? types(lanes, std::true_type{}) : types(lanes, std::false_type{}); };
    const int lanes = lanes_of(a.dim);
    if (lanes == 8) return pairs(std::integral_constant<int, 8>{});
    return lanes == 16 ? pairs(std::integral_constant<int, 16>{}) : pairs(std::integral_constant<int, 32>{});
}

}  // namespace

cudaError_t launch_rotary(const RotaryArgs& a, int num_sms, cudaStream_t stream) {
    return with_shape(a, [&](auto type, auto lanes, auto interleaved) {
        using T = decltype(type);
        constexpr int kLanes = decltype(lanes)::value, kRows = 32 / kLanes;
        constexpr bool kInterleaved = decltype(interleaved)::value;
        auto launch = [&](const void* fn, int iters) {
            auto chunks_of = [&](int heads) { return (heads + iters * kRows - 1) / (iters * kRows); };
            int chunks_q = chunks_of(a.heads[0]), chunks_k = chunks_of(a.heads[1]), chunks = chunks_q + chunks_k * (a.k_cache != nullptr ? 2 : 1);
            const int64_t ctas = (static_cast<int64_t>(a.tokens) * chunks * 32 + kRotaryThreads - 1) / kRotaryThreads;
            void* params[] = {const_cast<RotaryArgs*>(&a), &chunks_q, &chunks_k, &chunks};
            return launch_dependent(fn, dim3(static_cast<unsigned>(ctas)), dim3(kRotaryThreads), params, 0, stream);
        };
        // few rows: one at a time, on more warps
        const int64_t rows = static_cast<int64_t>(a.tokens) * (a.heads[0] + 2 * a.heads[1]);
        if (rows < static_cast<int64_t>(num_sms) * 16 * kRows * kForwardIters) return launch(reinterpret_cast<const void*>(rotary_kernel<T, kLanes, kInterleaved, 1>), 1);
        return launch(reinterpret_cast<const void*>(rotary_kernel<T, kLanes, kInterleaved, kForwardIters>), kForwardIters);
    });
}

int rotary_backward_ctas(const RotaryArgs& a, int num_sms) {
    const int heads_per_unit = kBackwardIters * 32 / lanes_of(a.dim);
    const int64_t units = static_cast<int64_t>(a.tokens) * ((a.heads[0] + heads_per_unit - 1) / heads_per_unit);
    return static_cast<int>(std::min<int64_t>((units * 32 + kRotaryThreads - 1) / kRotaryThreads, num_sms * 4));
}
cudaError_t launch_rotary_backward(const RotaryArgs& a, cudaStream_t stream) {
    void* params[] = {const_cast<RotaryArgs*>(&a)};
    const cudaError_t err = with_shape(a, [&](auto type, auto lanes, auto interleaved) {
        const void* fn = reinterpret_cast<const void*>(rotary_backward_kernel<decltype(type), decltype(lanes)::value, decltype(interleaved)::value, kBackwardIters>);
        return launch_dependent(fn, dim3(a.ctas), dim3(kRotaryThreads), params, 0, stream);
    });
    if (err != cudaSuccess) return err;
    return launch_dependent(reinterpret_cast<const void*>(rotary_reduce_kernel), dim3((2 * a.dim + 31) / 32), dim3(1024), params, 0, stream);
}

}  // namespace ep
