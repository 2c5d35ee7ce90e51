// Layer norm over the last axis and its gradients.
//
//     mean = sum x / H,  rstd = 1 / sqrt(sum (x - mean)^2 / H + eps),  xh = (x - mean) rstd,  y = xh w + b
//     g = dy w,  dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Values, statistics and sums are 32-bit; a result is rounded once to its type.
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace ep {

namespace {

template <class T>
__device__ __forceinline__ float to_float(T v) {
    if constexpr (sizeof(T) == 2) return __bfloat162float(v);
    else return v;
}
template <class T>
__device__ __forceinline__ T from_float(float v) {
    if constexpr (sizeof(T) == 2) return __float2bfloat16_rn(v);
    else return v;
}

// Two fp32 values in one register pair: Blackwell adds and multiplies both with one instruction, and these kernels would be bound by instruction issue
// without.
struct F2 {
    uint64_t v;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 unpack(F2 a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
    return r;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 mul_add(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ float mul_add(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float total(F2 a) {
    const float2 f = unpack(a);
    return f.x + f.y;
}
__device__ __forceinline__ float total(float a) { return a; }
template <class E>
__device__ __forceinline__ E both(float f) {
    if constexpr (std::is_same_v<E, F2>) return f2(f, f);
    else return f;
}

// A piece of kVec neighbouring values (16 bytes of a row, or one value where rows do not start on 16 bytes) as kN numbers or pairs of numbers
template <int kVec>
struct Piece {
    using E = std::conditional_t<kVec == 1, float, F2>;
    static constexpr int kN = kVec == 1 ? 1 : kVec / 2;
    E v[kN];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] = both<E>(0.f);
    }
    template <class T>
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kVec == 1) {
            v[0] = to_float(*p);
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < kVec / 4; ++i) {
                const float4 f = reinterpret_cast<const float4*>(p)[i];
                v[2 * i] = f2(f.x, f.y);
                v[2 * i + 1] = f2(f.z, f.w);
            }
        } else {
            uint32_t w[kVec / 2];
            if constexpr (kVec == 8) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
            else *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
#pragma unroll
            for (int i = 0; i < kVec / 2; ++i) v[i] = f2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        }
    }
    template <class T>
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (kVec == 1) {
            *p = from_float<T>(v[0]);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const float2 f = unpack(v[i]);
                if constexpr (sizeof(T) == 4) {
                    w[2 * i] = __float_as_uint(f.x);
                    w[2 * i + 1] = __float_as_uint(f.y);
                } else {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
                    w[i] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (kVec == 1) return v[0];
        else return i & 1 ? unpack(v[i / 2]).y : unpack(v[i / 2]).x;
    }
};
template <int kBytes>
__device__ __forceinline__ void copy_async(void* smem, const void* gmem) {
    if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ptx::smem_u32(smem)), "l"(gmem) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(ptx::smem_u32(smem)), "l"(gmem) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// Sums of kN (a power of two) values over a warp: in the first steps lanes trade values, so that half of them go on with half of the values.  Afterwards
// a lane has the sum of value lane / (32 / kN).
template <int kN>
__device__ __forceinline__ float warp_sums(float (&v)[kN]) {
    const int lane = threadIdx.x & 31;
    int o = 16;
#pragma unroll
    for (int n = kN; n > 1; n /= 2, o /= 2) {
        const bool upper = (lane & o) != 0;
#pragma unroll
        for (int i = 0; i < n / 2; ++i) {
            const float mine = upper ? v[i + n / 2] : v[i], other = upper ? v[i] : v[i + n / 2];
            v[i] = mine + __shfl_xor_sync(0xffffffffu, other, o);
        }
    }
#pragma unroll
    for (int r = 16 / kN; r > 0; r /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], r);
    return v[0];
}
// The same over the threads of a row, the sums on each of them.  Rows of a CTA: one barrier; `turn` picks one of two sets of shared words, so that the
// next sums may start while slower warps still read these.
template <int kN, bool kWarpRows>
__device__ __forceinline__ void row_sums(float (&v)[kN], float (*scratch)[32][kN], int& turn) {
    const int lane = threadIdx.x & 31;
    float sum = warp_sums<kN>(v);
    if constexpr (!kWarpRows) {
        float(*words)[kN] = scratch[turn];
        turn ^= 1;
        if (lane % (32 / kN) == 0) words[threadIdx.x >> 5][lane / (32 / kN)] = sum;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] = lane < static_cast<int>(blockDim.x >> 5) ? words[lane][i] : 0.f;
        sum = warp_sums<kN>(v);
    }
    if constexpr (kN == 1) {
        v[0] = sum;
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] = __shfl_sync(0xffffffffu, sum, i * (32 / kN));
    }
}

// As a piece lies in memory
template <class T, int kVec>
struct Raw {
    std::conditional_t<kVec == 1, T, uint4> v;
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kVec == 1) {
            v = *p;
        } else {
            const int4 q = ptx::ld_na_v4(p);
            v = make_uint4(q.x, q.y, q.z, q.w);
        }
    }
    __device__ __forceinline__ Piece<kVec> numbers() const {
        Piece<kVec> p;
        p.load(reinterpret_cast<const T*>(&v));
        return p;
    }
};

// The sum of one value per thread over a row, on each of its threads.  The warps' sums of a CTA's row lie in shared memory, zero where there is no warp, and every
// thread adds them up.
template <bool kWarpRows>
__device__ __forceinline__ float row_sum(float v, float4 (*words)[8], int& turn) {
    float one[1] = {v};
    float sum = warp_sums<1>(one);
    if constexpr (!kWarpRows) {
        float4* w = words[turn];
        turn ^= 1;
        if ((threadIdx.x & 31) == 0) reinterpret_cast<float*>(w)[threadIdx.x >> 5] = sum;
        __syncthreads();
        sum = 0.f;
        for (int i = 0; i < static_cast<int>(blockDim.x); i += 256) {
            const float4 p = w[i / 128], q = w[i / 128 + 1];
            sum += ((p.x + p.y) + (p.z + p.w)) + ((q.x + q.y) + (q.z + q.w));
        }
    }
    return sum;
}

// CTAs of `threads` that an SM should hold: 80 registers per thread for four pieces of 16 bytes (with 64, for more threads, they do not stay in registers)
constexpr int norm_min_ctas(int vec, int pieces, int threads) { return (vec == 1 ? (pieces == 8 ? 1024 : 512) : pieces < 4 || threads == 1024 ? 1024 : 768) / threads; }

// A row belongs to one warp (blockDim.y of them per CTA) or to a whole CTA; each thread has kPieces pieces of it in registers.  The registers that they came in take
// the next row's as soon as they have been made numbers.  Few threads per row: the two sums of a row are what it waits for, so an SM should
// have many rows under way, and shuffles and barriers cost by the warp.  8192 x 7168 bf16: 45 us, 5.2 TB/s (a copy of the same rows takes 39); 65536 x 512: 22 us, 6.2 TB/s.
// Making numbers of a row three times, from the registers that it came in, took 55 us and 64 registers; four CTAs of 64 registers spill: 57.
template <class T, class P, int kVec, int kPieces, bool kWarpRows, int kThreads>
__global__ void __launch_bounds__(kThreads, norm_min_ctas(kVec, kPieces, kThreads)) layer_norm_kernel(const LayerNormArgs a) {
    __shared__ float4 scratch[2][8];
    using E = typename Piece<kVec>::E;
    constexpr int kN = Piece<kVec>::kN;
    const int64_t first = blockIdx.x * blockDim.y + threadIdx.y, stride = static_cast<int64_t>(gridDim.x) * blockDim.y;
    const T* x = reinterpret_cast<const T*>(a.x);
    const P *w = reinterpret_cast<const P*>(a.weight), *b = reinterpret_cast<const P*>(a.bias);
    const float inverse = 1.f / a.hidden;
    const int col0 = threadIdx.x * kVec, step = blockDim.x * kVec;       // columns col0 + i * step
    if constexpr (!kWarpRows) {
        if (threadIdx.x < 16) scratch[threadIdx.x / 8][threadIdx.x % 8] = make_float4(0.f, 0.f, 0.f, 0.f);
        __syncthreads();
    }
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    Raw<T, kVec> raw[kPieces];
    if (first < a.rows)
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
            if (col0 + i * step < a.hidden) raw[i].load(x + first * a.ldx + col0 + i * step);
    int turn = 0;
    for (int64_t row = first; row < a.rows; row += stride) {
        Piece<kVec> p[kPieces];
        E acc[2] = {both<E>(0.f), both<E>(0.f)};
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
            if (col0 + i * step < a.hidden) {
                p[i] = raw[i].numbers();
#pragma unroll
                for (int j = 0; j < kN; ++j) acc[j & 1] = acc[j & 1] + p[i].v[j];
            }
        if (row + stride < a.rows)
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
                if (col0 + i * step < a.hidden) raw[i].load(x + (row + stride) * a.ldx + col0 + i * step);
        const float mean = row_sum<kWarpRows>(total(acc[0] + acc[1]), scratch, turn) * inverse;
        const E minus_mean = both<E>(-mean);
        acc[0] = acc[1] = both<E>(0.f);
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
            if (col0 + i * step < a.hidden) {
#pragma unroll
                for (int j = 0; j < kN; ++j) {
                    p[i].v[j] = p[i].v[j] + minus_mean;
                    acc[j & 1] = mul_add(p[i].v[j], p[i].v[j], acc[j & 1]);
                }
            }
        const float rstd = rsqrtf(row_sum<kWarpRows>(total(acc[0] + acc[1]), scratch, turn) * inverse + a.eps);
        const E scale = both<E>(rstd);
        T* y = reinterpret_cast<T*>(a.y) + row * a.hidden;
        auto finish = [&](auto with_bias) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int col = col0 + i * step;
                if (col < a.hidden) {
                    Piece<kVec> pw, pb;
                    pw.load(w + col);
                    if constexpr (decltype(with_bias)::value) pb.load(b + col);
#pragma unroll
                    for (int j = 0; j < kN; ++j) {
                        const E xh = p[i].v[j] * scale;
                        if constexpr (decltype(with_bias)::value) p[i].v[j] = mul_add(xh, pw.v[j], pb.v[j]);
                        else p[i].v[j] = xh * pw.v[j];
                    }
                    p[i].store(y + col);
                }
            }
        };
        if (b != nullptr) finish(std::true_type{});
        else finish(std::false_type{});
        if (threadIdx.x == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

// The gradients in one pass over x and dy: a row belongs to one warp (blockDim.y of them per CTA) or to a whole CTA, each thread has kValues values of it, and keeps
// its columns from row to row, so that the sums over the rows stay in registers; those of a CTA leave for a second kernel that adds them up in a fixed order.
// Rows come through shared memory, kStages - 1 ahead, each thread copying the pieces that it reads itself: one row ahead in registers leaves too few
// bytes in flight for HBM.  (Single bf16 values are read when they are needed.)  Bound by instruction issue and by the barrier that all warps of a wide row
// wait at: 8192 x 7168 bf16 78 us, 4.5 TB/s; 8192 x 4096 fp32 69 us, 5.8 TB/s.  Half as many registers for a second CTA of wide rows, with x, dy and the weights read
// from shared memory once more after the sums: 105 us.
__host__ __device__ constexpr int norm_stages(int size, int vec, int values) { return size * vec < 4 ? 0 : size * values >= 64 ? 3 : 4; }
template <class T, class P, int kVec, int kValues, bool kWarpRows, bool kBias>
__global__ void __launch_bounds__(kWarpRows ? 256 : kValues == 8 && kVec == 8 ? 896 : 512) layer_norm_backward_kernel(const LayerNormArgs a) {
    extern __shared__ __align__(16) uint8_t norm_smem[];
    __shared__ float scratch[2][32][2];
    using E = typename Piece<kVec>::E;
    constexpr int kN = Piece<kVec>::kN, kPieces = kValues / kVec, kBytes = sizeof(T) * kVec, kStages = norm_stages(sizeof(T), kVec, kValues);
    constexpr bool kAsync = kStages > 0;
    const int64_t first = blockIdx.x * blockDim.y + threadIdx.y, stride = static_cast<int64_t>(gridDim.x) * blockDim.y;
    const T *x = reinterpret_cast<const T*>(a.x), *dy = reinterpret_cast<const T*>(a.dy);
    const float inverse = 1.f / a.hidden;
    const int col0 = threadIdx.x * kVec, step = blockDim.x * kVec;       // columns col0 + i * step
    uint8_t* mine = norm_smem + (threadIdx.y * blockDim.x + threadIdx.x) * kBytes;
    const uint32_t pitch = blockDim.x * blockDim.y * kBytes;
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    auto request = [&](int stage, int64_t row) {
        if constexpr (kAsync) {
            if (row < a.rows)
#pragma unroll
                for (int i = 0; i < kPieces; ++i)
                    if (col0 + i * step < a.hidden) {
                        copy_async<kBytes>(mine + (stage * 2 * kPieces + i) * pitch, x + row * a.ldx + col0 + i * step);
                        copy_async<kBytes>(mine + ((stage * 2 + 1) * kPieces + i) * pitch, dy + row * a.lddy + col0 + i * step);
                    }
            copies_commit();
        }
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) request(s, first + s * stride);
    float next_mean = first < a.rows ? a.mean[first] : 0.f, next_rstd = first < a.rows ? a.rstd[first] : 0.f;
    Piece<kVec> pw[kPieces], dw[kPieces], db[kBias ? kPieces : 1];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        pw[i].clear();
        if (col0 + i * step < a.hidden) pw[i].load(reinterpret_cast<const P*>(a.weight) + col0 + i * step);
        dw[i].clear();
        if (kBias) db[i].clear();
    }
    int turn = 0, stage = 0;
    for (int64_t row = first; row < a.rows; row += stride) {
        const E minus_mean = both<E>(-next_mean), rstd = both<E>(next_rstd);
        if (row + stride < a.rows) {
            next_mean = a.mean[row + stride];
            next_rstd = a.rstd[row + stride];
        }
        if constexpr (kAsync) copies_wait<(kAsync ? kStages : 2) - 2>();
        Piece<kVec> xh[kPieces], g[kPieces];
        E acc_g = both<E>(0.f), acc_gx = both<E>(0.f);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            if (col0 + i * step < a.hidden) {
                if constexpr (kAsync) {
                    xh[i].load(reinterpret_cast<const T*>(mine + (stage * 2 * kPieces + i) * pitch));
                    g[i].load(reinterpret_cast<const T*>(mine + ((stage * 2 + 1) * kPieces + i) * pitch));
                } else {
                    xh[i].load(x + row * a.ldx + col0 + i * step);
                    g[i].load(dy + row * a.lddy + col0 + i * step);
                }
            } else {
                xh[i].clear();
                g[i].clear();          // dy, and with it all that follows, is zero where there is no column
            }
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                xh[i].v[j] = (xh[i].v[j] + minus_mean) * rstd;
                dw[i].v[j] = mul_add(g[i].v[j], xh[i].v[j], dw[i].v[j]);
                if (kBias) db[i].v[j] = db[i].v[j] + g[i].v[j];
                g[i].v[j] = g[i].v[j] * pw[i].v[j];
                acc_g = acc_g + g[i].v[j];
                acc_gx = mul_add(g[i].v[j], xh[i].v[j], acc_gx);
            }
        }
        float sum[2] = {total(acc_g), total(acc_gx)};
        row_sums<2, kWarpRows>(sum, scratch, turn);
        // (the stage that is filled now was read by this thread in the step before)
        if constexpr (kAsync) {
            request(stage == 0 ? kStages - 1 : stage - 1, row + (kStages - 1) * stride);
            stage = stage == kStages - 1 ? 0 : stage + 1;
        }
        const E minus_mg = both<E>(-sum[0] * inverse), minus_mgx = both<E>(-sum[1] * inverse);
        T* dx = reinterpret_cast<T*>(a.dx) + row * a.hidden;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
#pragma unroll
            for (int j = 0; j < kN; ++j) g[i].v[j] = mul_add(xh[i].v[j], minus_mgx, g[i].v[j] + minus_mg) * rstd;
            if (col0 + i * step < a.hidden) g[i].store(dx + col0 + i * step);
        }
    }
    const int width = (kBias ? 2 : 1) * a.hidden;
    float* part = a.partial + static_cast<int64_t>(blockIdx.x) * width;
    // (rows of a warp: the warps' sums one after the other through shared memory, where nobody reads rows any more)
    float* own = part;
    if constexpr (kWarpRows) {
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
        own = reinterpret_cast<float*>(norm_smem) + threadIdx.y * width;
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
        if (col0 + i * step < a.hidden)
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                own[col0 + i * step + j] = dw[i].get(j);
                if (kBias) own[a.hidden + col0 + i * step + j] = db[i].get(j);
            }
    if constexpr (kWarpRows) {
        __syncthreads();
        const float* all = reinterpret_cast<const float*>(norm_smem);
        for (int i = threadIdx.y * 32 + threadIdx.x; i < width; i += blockDim.y * 32) {
            float v = 0.f;
            for (int y = 0; y < static_cast<int>(blockDim.y); ++y) v += all[y * width + i];
            part[i] = v;
        }
    }
}

// Rows wider than a CTA's registers: passes over the row in memory (the later ones find it in L2).
constexpr int kWideThreads = 1024;
template <class T, class P>
__global__ void __launch_bounds__(kWideThreads) layer_norm_wide_kernel(const LayerNormArgs a) {
    __shared__ float scratch[2][32][1];
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const P *w = reinterpret_cast<const P*>(a.weight), *b = reinterpret_cast<const P*>(a.bias);
    int turn = 0;
    for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(a.x) + static_cast<int64_t>(row) * a.ldx;
        T* y = reinterpret_cast<T*>(a.y) + static_cast<int64_t>(row) * a.hidden;
        float sum[1] = {0.f};
        for (int i = threadIdx.x; i < a.hidden; i += kWideThreads) sum[0] += to_float(x[i]);
        row_sums<1, false>(sum, scratch, turn);
        const float mean = sum[0] / a.hidden;
        sum[0] = 0.f;
        for (int i = threadIdx.x; i < a.hidden; i += kWideThreads) {
            const float d = to_float(x[i]) - mean;
            sum[0] += d * d;
        }
        row_sums<1, false>(sum, scratch, turn);
        const float rstd = rsqrtf(sum[0] / a.hidden + a.eps);
        for (int i = threadIdx.x; i < a.hidden; i += kWideThreads) {
            const float v = (to_float(x[i]) - mean) * rstd * to_float(w[i]);
            y[i] = from_float<T>(b != nullptr ? v + to_float(b[i]) : v);
        }
        if (threadIdx.x == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}
template <class T, class P>
__global__ void __launch_bounds__(kWideThreads) layer_norm_backward_wide_kernel(const LayerNormArgs a) {
    __shared__ float scratch[2][32][2];
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const P* w = reinterpret_cast<const P*>(a.weight);
    float* part = a.partial + static_cast<int64_t>(blockIdx.x) * (a.db != nullptr ? 2 : 1) * a.hidden;
    int turn = 0;
    for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = reinterpret_cast<const T*>(a.x) + static_cast<int64_t>(row) * a.ldx, *dy = reinterpret_cast<const T*>(a.dy) + static_cast<int64_t>(row) * a.lddy;
        T* dx = reinterpret_cast<T*>(a.dx) + static_cast<int64_t>(row) * a.hidden;
        const float mean = a.mean[row], rstd = a.rstd[row];
        const bool start = row == static_cast<int>(blockIdx.x);
        float sum[2] = {0.f, 0.f};
        for (int i = threadIdx.x; i < a.hidden; i += kWideThreads) {
            const float d = to_float(dy[i]), xh = (to_float(x[i]) - mean) * rstd, g = d * to_float(w[i]);
            sum[0] += g;
            sum[1] += g * xh;
            part[i] = (start ? 0.f : part[i]) + d * xh;
            if (a.db != nullptr) part[a.hidden + i] = (start ? 0.f : part[a.hidden + i]) + d;
        }
        row_sums<2, false>(sum, scratch, turn);
        const float mg = sum[0] / a.hidden, mgx = sum[1] / a.hidden;
        for (int i = threadIdx.x; i < a.hidden; i += kWideThreads)
            dx[i] = from_float<T>(rstd * (to_float(dy[i]) * to_float(w[i]) - mg - (to_float(x[i]) - mean) * rstd * mgx));
    }
}

// d_weight and d_bias: 32 columns per CTA, the slices shared out over 32 warps
constexpr int kReduceWarps = 32;
template <class P>
__global__ void __launch_bounds__(kReduceWarps * 32) layer_norm_reduce_kernel(const LayerNormArgs a) {
    __shared__ float sums[kReduceWarps][33];
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + lane, width = static_cast<int64_t>(a.db != nullptr ? 2 : 1) * a.hidden;
    float v = 0.f;
    if (col < width)
        for (int s0 = warp; s0 < a.slices; s0 += 8 * kReduceWarps) {        // eight requested at once
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = s0 + i * kReduceWarps < a.slices ? a.partial[(s0 + i * kReduceWarps) * width + col] : 0.f;
            v += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        }
    sums[warp][lane] = v;
    __syncthreads();
    v = sums[lane][warp];          // column `warp`, slice group `lane`
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int64_t out = static_cast<int64_t>(blockIdx.x) * 32 + warp;
    if (lane == 0 && out < width) {
        if (out < a.hidden) reinterpret_cast<P*>(a.dw)[out] = from_float<P>(v);
        else reinterpret_cast<P*>(a.db)[out - a.hidden] = from_float<P>(v);
    }
}

using NormKernel = void (*)(LayerNormArgs);
template <class T, class P>
NormKernel forward_kernel(const NormShape& n) {
    constexpr int kVec = 16 / sizeof(T);
    if (n.values == 0) return layer_norm_wide_kernel<T, P>;
    if (n.vec == 1) {
        if (n.values == 8) return n.warp_rows ? layer_norm_kernel<T, P, 1, 8, true, 256> : layer_norm_kernel<T, P, 1, 8, false, 512>;
        return layer_norm_kernel<T, P, 1, 16, false, 512>;
    }
    if (n.warp_rows && n.values == kVec) return layer_norm_kernel<T, P, kVec, 1, true, 256>;
    if (n.warp_rows) return n.values == 2 * kVec ? layer_norm_kernel<T, P, kVec, 2, true, 256> : layer_norm_kernel<T, P, kVec, 4, true, 256>;
    if (n.threads <= 256) return layer_norm_kernel<T, P, kVec, 4, false, 256>;
    return n.threads <= 384 ? layer_norm_kernel<T, P, kVec, 4, false, 384> : layer_norm_kernel<T, P, kVec, 4, false, 1024>;
}
NormKernel forward_kernel(const LayerNormArgs& a, const NormShape& n) {
    if (a.x_bf16) return a.param_bf16 ? forward_kernel<__nv_bfloat16, __nv_bfloat16>(n) : forward_kernel<__nv_bfloat16, float>(n);
    return a.param_bf16 ? forward_kernel<float, __nv_bfloat16>(n) : forward_kernel<float, float>(n);
}
template <class T, class P, int kVec, int kValues, bool kWarpRows>
NormKernel backward_kernel(bool bias) {
    return bias ? layer_norm_backward_kernel<T, P, kVec, kValues, kWarpRows, true> : layer_norm_backward_kernel<T, P, kVec, kValues, kWarpRows, false>;
}
template <class T, class P, int kVec>
NormKernel backward_kernel(const NormShape& n, bool bias) {
    if (n.warp_rows) return n.values == 8 ? backward_kernel<T, P, kVec, 8, true>(bias) : backward_kernel<T, P, kVec, 16, true>(bias);
    if constexpr (kVec != 4)
        if (n.values == 8) return backward_kernel<T, P, kVec, 8, false>(bias);
    return backward_kernel<T, P, kVec, 16, false>(bias);
}
template <class T, class P>
NormKernel backward_kernel(const NormShape& n, bool bias) {
    if (n.values == 0) return layer_norm_backward_wide_kernel<T, P>;
    return n.vec == 1 ? backward_kernel<T, P, 1>(n, bias) : backward_kernel<T, P, 16 / sizeof(T)>(n, bias);
}
NormKernel backward_kernel(const LayerNormArgs& a, const NormShape& n, bool bias) {
    if (a.x_bf16) return a.param_bf16 ? backward_kernel<__nv_bfloat16, __nv_bfloat16>(n, bias) : backward_kernel<__nv_bfloat16, float>(n, bias);
    return a.param_bf16 ? backward_kernel<float, __nv_bfloat16>(n, bias) : backward_kernel<float, float>(n, bias);
}
bool on_16_bytes(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// At most `ctas` CTAs, as many as fit on the SMs.  Not asked for where every CTA has an SM: that would be a tenth of what a small call takes.
int resident_ctas(const void* fn, int threads, int smem, int64_t ctas, int num_sms) {
    int n = 1;
    if (ctas > num_sms) allow_shared_memory(fn, threads, smem, &n);      // (what fails here fails again, and is reported, at the launch)
    return static_cast<int>(std::min<int64_t>(ctas, static_cast<int64_t>(n) * num_sms));
}

bool rows_on_16_bytes(const LayerNormArgs& a, bool backward) {
    const int size = a.x_bf16 ? 2 : 4;
    return static_cast<int64_t>(a.hidden) * size % 16 == 0 && a.ldx * size % 16 == 0 && on_16_bytes(a.x) && on_16_bytes(a.weight) && (a.bias == nullptr || on_16_bytes(a.bias)) &&
           (!backward || (a.lddy * size % 16 == 0 && on_16_bytes(a.dy)));
}

cudaError_t launch_rows(const void* fn, const NormShape& n, void** params, cudaStream_t stream) {
    if (n.smem > 40 * 1024) {      // (48 KB with the static one need no leave)
        const cudaError_t err = allow_shared_memory(fn, n.threads * n.rows_per_cta, n.smem, nullptr);
        if (err != cudaSuccess) return err;
    }
    return launch_dependent(fn, dim3(n.ctas), dim3(n.threads, n.rows_per_cta), params, n.smem, stream);
}

}  // namespace

// Pieces of 16 bytes where every row of every operand starts on 16 bytes, single values otherwise.  Four pieces (eight or sixteen values) per thread, so that a row has few
// threads; one or two where those make do with a warp.
cudaError_t launch_layer_norm(const LayerNormArgs& args, int num_sms, cudaStream_t stream) {
    if (args.hidden < 1 || args.rows < 0) return cudaErrorInvalidValue;
    if (args.rows == 0) return cudaSuccess;
    LayerNormArgs a = args;
    NormShape n{};
    n.vec = rows_on_16_bytes(a, false) ? 16 / (a.x_bf16 ? 2 : 4) : 1;
    n.values = n.vec == 1 ? (a.hidden <= 8 * 512 ? 8 : 16) : a.hidden <= 32 * n.vec ? n.vec : a.hidden <= 64 * n.vec ? 2 * n.vec : 4 * n.vec;
    n.threads = static_cast<int>((static_cast<int64_t>(a.hidden) + n.values - 1) / n.values + 31) / 32 * 32;
    n.warp_rows = n.threads == 32;
    n.rows_per_cta = n.warp_rows ? 8 : 1;
    if (n.threads > (n.vec == 1 ? 512 : 1024)) {
        n.values = 0;
        n.threads = kWideThreads;
    }
    const void* fn = reinterpret_cast<const void*>(forward_kernel(a, n));
    const int64_t ctas = (static_cast<int64_t>(a.rows) + n.rows_per_cta - 1) / n.rows_per_cta;
    n.ctas = resident_ctas(fn, n.threads * n.rows_per_cta, 0, ctas, num_sms);
    void* params[] = {&a};
    return launch_rows(fn, n, params, stream);
}

// Backward: pieces of 16 bytes where every row of every operand starts on 16 bytes, single values otherwise.  A warp per row up to 512 channels, then a CTA of up to
// 512 threads with sixteen values of a row each (128 registers); wider rows stay in memory.  bf16 rows that leave room for one such CTA on an SM take eight values on up to
// 896 threads: 8192 x 7168 78 us, with sixteen 82; 16384 x 4096 101 / 81, 32768 x 2048 87 / 78.  So do single values
// up to 4096 channels.
// (Whether there is a bias changes nothing, so that the weights' gradient has the same bits with and without.)
NormShape layer_norm_backward_shape(const LayerNormArgs& a, int num_sms) {
    NormShape n{};
    const int size = a.x_bf16 ? 2 : 4;
    n.vec = rows_on_16_bytes(a, true) ? 16 / size : 1;
    n.warp_rows = a.hidden <= 512;
    n.values = a.hidden <= 256 || (n.vec == 8 && a.hidden > 16 * 256 && a.hidden <= 8 * 896) || (n.vec == 1 && a.hidden > 512 && a.hidden <= 8 * 512) ? 8 : a.hidden <= 16 * 512 ? 16 : 0;
    n.threads = n.values == 0 ? kWideThreads : n.warp_rows ? 32 : ((a.hidden + n.values - 1) / n.values + 31) / 32 * 32;
    n.rows_per_cta = n.warp_rows ? 8 : 1;
    n.smem = norm_stages(size, n.vec, n.values) * 2 * n.values * size * n.threads * n.rows_per_cta;
    if (n.warp_rows) n.smem = std::max(n.smem, n.rows_per_cta * 2 * a.hidden * 4);
    // every slice of the gradient's sums costs a row of 32-bit values written and read again: at least four rows share one
    int64_t ctas = (static_cast<int64_t>(a.rows) + n.rows_per_cta - 1) / n.rows_per_cta;
    ctas = std::min<int64_t>(ctas, std::max<int64_t>(num_sms, a.rows / 4));
    n.ctas = std::max(1, resident_ctas(reinterpret_cast<const void*>(backward_kernel(a, n, true)), n.threads * n.rows_per_cta, n.smem, ctas, num_sms));
    return n;
}

cudaError_t launch_layer_norm_backward(const LayerNormArgs& args, const NormShape& n, cudaStream_t stream) {
    if (args.hidden < 1 || args.rows < 0) return cudaErrorInvalidValue;
    LayerNormArgs a = args;
    a.slices = a.rows > 0 ? n.ctas : 0;
    void* params[] = {&a};
    if (a.rows > 0) {
        const cudaError_t err = launch_rows(reinterpret_cast<const void*>(backward_kernel(a, n, a.db != nullptr)), n, params, stream);
        if (err != cudaSuccess) return err;
    }
    const int64_t width = static_cast<int64_t>(a.db != nullptr ? 2 : 1) * a.hidden;
    return launch_dependent(a.param_bf16 ? reinterpret_cast<const void*>(layer_norm_reduce_kernel<__nv_bfloat16>) : reinterpret_cast<const void*>(layer_norm_reduce_kernel<float>),
                            dim3(static_cast<unsigned>((width + 31) / 32)), dim3(kReduceWarps * 32), params, 0, stream);
}

}  // namespace ep
