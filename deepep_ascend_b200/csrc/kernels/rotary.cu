// RMS norm of every query and key head and rotation of its channels by the token's position, in one pass, and its gradient.  Per head x of D channels, with the weight w:
//
//     rstd = (mean x^2 + eps)^-1/2,   n = rstd x w,   (a, b) of a pair of channels -> (a cos - b sin, b cos + a sin)
//
// where the pairs are channels (i, i + R/2) of the first R channels, or, interleaved, (2 i, 2 i + 1).  Backwards: g = dy rotated back,
//
//     dw = sum over tokens and heads of g rstd x,     u = g w,     dx = rstd (u - rstd^2 x mean(u x))
//
// Bound by memory: every value is read once and written once.  A row of D channels lies on 8, 16 or 32 lanes of a warp, eight channels each: neighbours where pairs are neighbours,
// else four and their partners, so that no lane asks another for them (eight neighbours, and their partners' values by shuffles: 3 us more for 8192 x 64 heads of 128).  What 16-bit heads take beyond that is instruction issue,
// so values go in pairs and 1/sqrt is CUDA's of 2 ulp (the one that rounds to nearest: 59 instead of 54 us).
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace ep {

namespace {

using bf16 = __nv_bfloat16;
constexpr int kRotaryThreads = 256;
// Rows of a lane group that a warp has at once, and CTAs of an SM: what is on its way at a time.  8192 x 64 heads of 128, bf16: 54 us (three CTAs: 62; two rows: 8 us more, eight
// on three CTAs: 7 more, two times four behind one another: 10 more, by the registers that they take from the loads); gradients 91 (two rows: 7 more, three CTAs: 15 more), where four rows of 32-bit values do not fit the registers (4096 x 40 heads: 86 us instead of 48).
constexpr int kForwardIters = 4, kForwardCtas = 4, kBackwardCtas = 2;
__host__ __device__ constexpr int backward_iters(int value_bytes) { return value_bytes == 2 ? 4 : 2; }

// Two values at once
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ float both(uint64_t v) {
    float a, b;
    unpair(v, a, b);
    return a + b;
}

// Eight channels, four from lo on and four from hi on (kWhole: neighbours)
template <class T>
struct Eight {
    uint4 raw[sizeof(T) / 2];
};
template <bool kWhole, class T>
__device__ __forceinline__ Eight<T> load8(const T* p, int lo, int hi) {
    Eight<T> e;
    if constexpr (sizeof(T) == 4) {
        e.raw[0] = *reinterpret_cast<const uint4*>(p + lo);
        e.raw[1] = *reinterpret_cast<const uint4*>(p + (kWhole ? lo + 4 : hi));
    } else if constexpr (kWhole) {
        e.raw[0] = *reinterpret_cast<const uint4*>(p + lo);
    } else {
        const uint2 a = *reinterpret_cast<const uint2*>(p + lo), b = *reinterpret_cast<const uint2*>(p + hi);
        e.raw[0] = make_uint4(a.x, a.y, b.x, b.y);
    }
    return e;
}
template <bool kWhole, class T>
__device__ __forceinline__ void store8(T* p, int lo, int hi, const Eight<T>& e) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<uint4*>(p + lo) = e.raw[0];
        *reinterpret_cast<uint4*>(p + (kWhole ? lo + 4 : hi)) = e.raw[1];
    } else if constexpr (kWhole) {
        *reinterpret_cast<uint4*>(p + lo) = e.raw[0];
    } else {
        *reinterpret_cast<uint2*>(p + lo) = make_uint2(e.raw[0].x, e.raw[0].y);
        *reinterpret_cast<uint2*>(p + hi) = make_uint2(e.raw[0].z, e.raw[0].w);
    }
}
__device__ __forceinline__ void to_float(const Eight<bf16>& e, uint64_t (&f)[4]) {
    const uint32_t w[4] = {e.raw[0].x, e.raw[0].y, e.raw[0].z, e.raw[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
__device__ __forceinline__ void to_float(const Eight<float>& e, uint64_t (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        f[2 * i] = pair(__uint_as_float(e.raw[i].x), __uint_as_float(e.raw[i].y));
        f[2 * i + 1] = pair(__uint_as_float(e.raw[i].z), __uint_as_float(e.raw[i].w));
    }
}
template <class T>
__device__ __forceinline__ Eight<T> from_float(const uint64_t (&f)[4]) {
    Eight<T> e;
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) unpair(f[i], v[2 * i], v[2 * i + 1]);
    if constexpr (sizeof(T) == 2) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
        e.raw[0] = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) e.raw[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
    }
    return e;
}
template <class T>
__device__ __forceinline__ Eight<T> all_of(float x) {
    const uint64_t v[4] = {pair(x, x), pair(x, x), pair(x, x), pair(x, x)};
    return from_float<T>(v);
}
// ... of the partners of a lane's channels
template <bool kInterleaved>
__device__ __forceinline__ uint64_t partner_of(const uint64_t (&v)[4], int i) {
    if constexpr (kInterleaved) {
        float a, b;
        unpair(v[i], a, b);
        return pair(b, a);
    } else {
        return v[i ^ 2];
    }
}
template <bool kWhole>
__device__ __forceinline__ void load_weight(const void* w, int is_bf16, int lo, int hi, uint64_t (&f)[4]) {
    if (is_bf16) to_float(load8<kWhole>(static_cast<const bf16*>(w), lo, hi), f);
    else to_float(load8<kWhole>(static_cast<const float*>(w), lo, hi), f);
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
    static constexpr int kRows = 32 / kLanes;            // of a warp
    int sub, lo, hi, angle;                              // row of the warp, channels, first angle
    bool on, turned;                                     // lanes that hold channels, that hold rotated ones
    __device__ __forceinline__ Place(int dim, int rotary) {
        const int lane = threadIdx.x & 31, in = lane % kLanes;
        sub = lane / kLanes;
        on = in * 8 < dim;
        turned = in * 8 < rotary;
        lo = kInterleaved || !turned ? in * 8 : in * 4;
        hi = kInterleaved || !turned ? lo + 4 : rotary / 2 + lo;
        angle = in * 4;
    }
    __device__ __forceinline__ int channel(int j) const { return j < 4 ? lo + j : hi + j - 4; }
};
// What a lane's eight channels take of themselves and of their partners: cosines and signed sines, or these times the channels' weights.  Rows of zeros in front of the
// table, of no numbers behind it.
template <bool kInterleaved>
struct Angles {
    uint64_t own[4], partner[4];
    float keep;
    template <class P>
    __device__ __forceinline__ Angles(const RotaryArgs& a, const P& place, int64_t position) {
        keep = position < 0 ? 0.f : (position < a.num_positions ? 1.f : __int_as_float(0x7fc00000));
        const float* row = a.table + (position >= 0 && position < a.num_positions ? position : 0) * a.rotary + place.angle;
        const bool read = place.turned && a.num_positions > 0;
        const float4 c = read ? *reinterpret_cast<const float4*>(row) : make_float4(1.f, 1.f, 1.f, 1.f);
        const float4 s = read ? *reinterpret_cast<const float4*>(row + a.rotary / 2) : make_float4(0.f, 0.f, 0.f, 0.f);
        if constexpr (kInterleaved) {
            own[0] = pair(c.x, c.x), own[1] = pair(c.y, c.y), own[2] = pair(c.z, c.z), own[3] = pair(c.w, c.w);
            partner[0] = pair(-s.x, s.x), partner[1] = pair(-s.y, s.y), partner[2] = pair(-s.z, s.z), partner[3] = pair(-s.w, s.w);
        } else {
            own[0] = own[2] = pair(c.x, c.y), own[1] = own[3] = pair(c.z, c.w);
            partner[0] = pair(-s.x, -s.y), partner[1] = pair(-s.z, -s.w), partner[2] = pair(s.x, s.y), partner[3] = pair(s.z, s.w);
        }
    }
    __device__ __forceinline__ void times(const uint64_t (&w)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            own[i] = mul2(own[i], w[i]);
            partner[i] = mul2(partner[i], partner_of<kInterleaved>(w, i));
        }
    }
    // (the other way round: the sines' signs)
    __device__ __forceinline__ void back() {
#pragma unroll
        for (int i = 0; i < 4; ++i) partner[i] ^= 0x8000000080000000ull;
    }
};

// Rows [kIters] of a warp: heads of one kind (queries, keys, values) of one token
template <class T, int kLanes, bool kInterleaved, int kIters>
__global__ void __launch_bounds__(kRotaryThreads, kForwardCtas) rotary_kernel(const __grid_constant__ RotaryArgs a, int chunks_q, int chunks_k, int chunks) {
    using Lane = Place<kLanes, kInterleaved>;
    constexpr int kHeads = kIters * Lane::kRows;
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const uint32_t unit = blockIdx.x * (kRotaryThreads / 32) + (threadIdx.x >> 5);      // (fewer than 2^32)
    const int64_t token = unit / static_cast<uint32_t>(chunks);
    if (token >= a.tokens) return;
    int chunk = static_cast<int>(unit - static_cast<uint32_t>(token) * chunks);
    const int kind = chunk < chunks_q ? 0 : (chunk < chunks_q + chunks_k ? 1 : 2);
    chunk -= kind == 0 ? 0 : (kind == 1 ? chunks_q : chunks_q + chunks_k);
    const Lane place(a.dim, a.rotary);
    const float inv_dim = 1.f / a.dim;
    const HeadsView& x = kind == 2 ? a.v : a.x[kind];
    const int heads = a.heads[kind == 0 ? 0 : 1], head0 = chunk * kHeads + place.sub;
    const int64_t position = kind == 2 ? 0 : load_index(a.positions, a.positions_64, token);
    Eight<T> raw[kIters] = {};
#pragma unroll
    for (int i = 0; i < kIters; ++i)
        if (place.on && head0 + i * Lane::kRows < heads)
            raw[i] = load8<kInterleaved>(static_cast<const T*>(x.data) + token * x.stride_token + (head0 + i * Lane::kRows) * x.stride_head, place.lo, place.hi);
    T *out, *too = nullptr;                              // (keys may go to a cache and to a result)
    int64_t pitch;
    bool write = place.on;
    if (kind == 0 || !a.append) {
        out = static_cast<T*>(a.out[kind]) + token * heads * a.dim;
        pitch = a.dim;
    } else {
        const int64_t slot = load_index(a.slots, a.slots_64, token);
        write = write && slot >= 0 && slot < a.num_slots;
        const int64_t page = slot / a.page_size;
        out = static_cast<T*>(kind == 1 ? a.k_cache : a.v_cache) + page * a.stride_page + (slot - page * a.page_size) * a.stride_slot;
        pitch = a.stride_head;
        if (kind == 1 && a.out[1] != nullptr) too = static_cast<T*>(a.out[1]) + (token * heads + head0) * a.dim;
    }
    if (kind == 2) {
#pragma unroll
        for (int i = 0; i < kIters; ++i)
            if (write && head0 + i * Lane::kRows < heads) store8<kInterleaved>(out + (head0 + i * Lane::kRows) * pitch, place.lo, place.hi, raw[i]);
        return;
    }
    uint64_t w[4] = {};
    if (place.on) load_weight<kInterleaved>(a.weight[kind], a.param_bf16, place.lo, place.hi, w);
    Angles<kInterleaved> turn(a, place, position);
    out += head0 * pitch;
    if (turn.keep != 1.f) {
        const Eight<T> fill = all_of<T>(turn.keep);
#pragma unroll
        for (int i = 0; i < kIters; ++i)
            if (head0 + i * Lane::kRows < heads) {
                if (write) store8<kInterleaved>(out + i * Lane::kRows * pitch, place.lo, place.hi, fill);
                if (too != nullptr && place.on) store8<kInterleaved>(too + i * Lane::kRows * a.dim, place.lo, place.hi, fill);
            }
        return;
    }
    turn.times(w);
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
        uint64_t v[4], squares = 0;
        to_float(raw[i], v);
#pragma unroll
        for (int j = 0; j < 4; ++j) squares = fma2(v[j], v[j], squares);
        const float rstd = rsqrtf(sum_row<kLanes>(both(squares)) * inv_dim + a.eps);
        const uint64_t rstd2 = pair(rstd, rstd);
        uint64_t y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = mul2(rstd2, fma2(partner_of<kInterleaved>(v, j), turn.partner[j], mul2(v[j], turn.own[j])));
        if (head0 + i * Lane::kRows < heads) {
            const Eight<T> e = from_float<T>(y);
            if (write) store8<kInterleaved>(out + i * Lane::kRows * pitch, place.lo, place.hi, e);
            if (too != nullptr && place.on) store8<kInterleaved>(too + i * Lane::kRows * a.dim, place.lo, place.hi, e);
        }
    }
}

// Gradient: a warp takes chunks of heads, those of queries and then those of keys, and keeps its sums of the weight's gradient
template <class T, int kLanes, bool kInterleaved, int kIters>
__global__ void __launch_bounds__(kRotaryThreads, kBackwardCtas) rotary_backward_kernel(const __grid_constant__ RotaryArgs a) {
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
        uint64_t w[4] = {}, dw[4] = {};
        if (place.on) load_weight<kInterleaved>(a.weight[kind], a.param_bf16, place.lo, place.hi, w);
        // neighbouring chunks, the next one's values on their way while this one's are worked on
        const int64_t warps = static_cast<int64_t>(gridDim.x) * kWarps, share = (units + warps - 1) / warps;
        const int64_t begin = (static_cast<int64_t>(blockIdx.x) * kWarps + warp) * share, end = min(begin + share, units);
        Eight<T> x[kIters] = {}, d[kIters] = {}, next_x[kIters] = {}, next_d[kIters] = {};
        int64_t token = begin / max(chunks, 1), next_token = token;      // (no chunks: no heads of this kind)
        int chunk = static_cast<int>(begin - token * chunks), next_chunk = chunk;
        auto request = [&]() {
#pragma unroll
            for (int i = 0; i < kIters; ++i) {
                const int64_t head = next_chunk * kHeads + place.sub + i * Lane::kRows;
                next_x[i] = next_d[i] = Eight<T>{};
                if (place.on && head < heads) {
                    next_x[i] = load8<kInterleaved>(static_cast<const T*>(a.x[kind].data) + next_token * a.x[kind].stride_token + head * a.x[kind].stride_head, place.lo, place.hi);
                    next_d[i] = load8<kInterleaved>(static_cast<const T*>(a.dy[kind].data) + next_token * a.dy[kind].stride_token + head * a.dy[kind].stride_head, place.lo, place.hi);
                }
            }
        };
        if (begin < end) request();
#pragma unroll 1
        for (int64_t unit = begin; unit < end; ++unit) {
            token = next_token;
            chunk = next_chunk;
#pragma unroll
            for (int i = 0; i < kIters; ++i) x[i] = next_x[i], d[i] = next_d[i];
            if (++next_chunk == chunks) next_chunk = 0, ++next_token;
            if (unit + 1 < end) request();
            const int head0 = chunk * kHeads + place.sub;
            Angles<kInterleaved> turn(a, place, load_index(a.positions, a.positions_64, token));
            turn.back();
            T* out = static_cast<T*>(a.out[kind]) + (token * heads + head0) * a.dim;
            if (turn.keep != 1.f) {
                const Eight<T> fill = all_of<T>(turn.keep);
#pragma unroll
                for (int i = 0; i < kIters; ++i)
                    if (place.on && head0 + i * Lane::kRows < heads) store8<kInterleaved>(out + i * Lane::kRows * a.dim, place.lo, place.hi, fill);
                if (turn.keep != 0.f)
#pragma unroll
                    for (int j = 0; j < 4; ++j) dw[j] = pair(turn.keep, turn.keep);
                continue;
            }
#pragma unroll
            for (int i = 0; i < kIters; ++i) {
                // (rows that are not there are zeros)
                uint64_t v[4], g[4], own[4], squares = 0, along = 0;
                to_float(x[i], v);
                to_float(d[i], own);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    g[j] = fma2(partner_of<kInterleaved>(own, j), turn.partner[j], mul2(own[j], turn.own[j]));
                    squares = fma2(v[j], v[j], squares);
                    along = fma2(mul2(g[j], w[j]), v[j], along);
                }
                const float mean = sum_row<kLanes>(both(squares)) * inv_dim, with = sum_row<kLanes>(both(along)) * inv_dim;
                const float rstd = rsqrtf(mean + a.eps), back = -rstd * rstd * rstd * with;
                const bool there = head0 + i * Lane::kRows < heads;
                const uint64_t rstd2 = pair(rstd, rstd), back2 = pair(back, back);
                uint64_t dx[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint64_t gr = mul2(g[j], rstd2);
                    dx[j] = fma2(gr, w[j], mul2(v[j], back2));
                    dw[j] = fma2(gr, v[j], dw[j]);
                }
                if (there && place.on) store8<kInterleaved>(out + i * Lane::kRows * a.dim, place.lo, place.hi, from_float<T>(dx));
            }
        }
        float sums[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) unpair(dw[j], sums[2 * j], sums[2 * j + 1]);
        // rows of a warp, then warps
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int o = kLanes; o < 32; o <<= 1) sums[j] += __shfl_xor_sync(0xffffffffu, sums[j], o);
        __syncthreads();
        if (place.sub == 0)
#pragma unroll
            for (int j = 0; j < 8; ++j) s_sum[warp][place.on ? place.channel(j) : place.lo + j] = sums[j];
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
            int chunks_q = chunks_of(a.heads[0]), chunks_k = chunks_of(a.heads[1]), chunks = chunks_q + chunks_k * (a.append ? 2 : 1);
            const int64_t ctas = (static_cast<int64_t>(a.tokens) * chunks * 32 + kRotaryThreads - 1) / kRotaryThreads;
            void* params[] = {const_cast<RotaryArgs*>(&a), &chunks_q, &chunks_k, &chunks};
            return launch_dependent(fn, dim3(static_cast<unsigned>(ctas)), dim3(kRotaryThreads), params, 0, stream);
        };
        // few rows: one at a time, on more warps
        const int64_t rows = static_cast<int64_t>(a.tokens) * (a.heads[0] + 2 * a.heads[1]);
        if (rows < static_cast<int64_t>(num_sms) * 32 * kRows * kForwardIters) return launch(reinterpret_cast<const void*>(rotary_kernel<T, kLanes, kInterleaved, 1>), 1);
        return launch(reinterpret_cast<const void*>(rotary_kernel<T, kLanes, kInterleaved, kForwardIters>), kForwardIters);
    });
}

int rotary_backward_ctas(const RotaryArgs& a, int num_sms) {
    const int heads_per_unit = backward_iters(a.x_bf16 ? 2 : 4) * 32 / lanes_of(a.dim);
    const int64_t units = std::max<int64_t>(static_cast<int64_t>(a.tokens) * ((std::max(a.heads[0], a.heads[1]) + heads_per_unit - 1) / heads_per_unit), 1);
    return static_cast<int>(std::min<int64_t>((units * 32 + kRotaryThreads - 1) / kRotaryThreads, num_sms * kBackwardCtas));
}
cudaError_t launch_rotary_backward(const RotaryArgs& a, cudaStream_t stream) {
    void* params[] = {const_cast<RotaryArgs*>(&a)};
    const cudaError_t err = with_shape(a, [&](auto type, auto lanes, auto interleaved) {
        const void* fn = reinterpret_cast<const void*>(rotary_backward_kernel<decltype(type), decltype(lanes)::value, decltype(interleaved)::value, backward_iters(sizeof(type))>);
        return launch_dependent(fn, dim3(a.ctas), dim3(kRotaryThreads), params, 0, stream);
    });
    if (err != cudaSuccess) return err;
    return launch_dependent(reinterpret_cast<const void*>(rotary_reduce_kernel), dim3((2 * a.dim + 31) / 32), dim3(1024), params, 0, stream);
}

}  // namespace ep
