// Layer norm over the last axis and its gradients.
//
//     mean = sum x / H,  rstd = 1 / sqrt(sum (x - mean)^2 / H + eps),  xh = (x - mean) rstd,  y = xh w + b
//     g = dy w,  dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Values, statistics and sums are 32-bit; a result is rounded once to its type.
#include <algorithm>

#include "common.cuh"

namespace ep {

namespace {

constexpr int kNormThreads = 256;

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

// sums of two values over the CTA, the same on every thread; `scratch` may be used again after the next barrier
__device__ __forceinline__ float2 block_sum(float a, float b, float2* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    __syncthreads();
    if (lane == 0) scratch[warp] = make_float2(a, b);
    __syncthreads();
    a = b = 0.f;
    for (int w = 0; w < warps; ++w) {
        a += scratch[w].x;
        b += scratch[w].y;
    }
    return make_float2(a, b);
}

template <class T, class P>
__global__ void __launch_bounds__(kNormThreads) layer_norm_kernel(const LayerNormArgs a) {
    __shared__ float2 scratch[32];
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const T* x = reinterpret_cast<const T*>(a.x) + static_cast<int64_t>(blockIdx.x) * a.ldx;
    T* y = reinterpret_cast<T*>(a.y) + static_cast<int64_t>(blockIdx.x) * a.hidden;
    const P *w = reinterpret_cast<const P*>(a.weight), *b = reinterpret_cast<const P*>(a.bias);
    float sum = 0.f, sq = 0.f;
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x) sum += to_float(x[i]);
    const float mean = block_sum(sum, 0.f, scratch).x / a.hidden;
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x) {
        const float d = to_float(x[i]) - mean;
        sq += d * d;
    }
    const float rstd = 1.f / sqrtf(block_sum(sq, 0.f, scratch).x / a.hidden + a.eps);
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x) {
        const float v = (to_float(x[i]) - mean) * rstd * to_float(w[i]);
        y[i] = from_float<T>(b != nullptr ? v + to_float(b[i]) : v);
    }
    if (threadIdx.x == 0) {
        a.mean[blockIdx.x] = mean;
        a.rstd[blockIdx.x] = rstd;
    }
}

template <class T, class P>
__global__ void __launch_bounds__(kNormThreads) layer_norm_dx_kernel(const LayerNormArgs a) {
    __shared__ float2 scratch[32];
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const int64_t row = blockIdx.x;
    const T *x = reinterpret_cast<const T*>(a.x) + row * a.ldx, *dy = reinterpret_cast<const T*>(a.dy) + row * a.lddy;
    T* dx = reinterpret_cast<T*>(a.dx) + row * a.hidden;
    const P* w = reinterpret_cast<const P*>(a.weight);
    const float mean = a.mean[row], rstd = a.rstd[row];
    float sg = 0.f, sgx = 0.f;
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x) {
        const float g = to_float(dy[i]) * to_float(w[i]);
        sg += g;
        sgx += g * ((to_float(x[i]) - mean) * rstd);
    }
    const float2 s = block_sum(sg, sgx, scratch);
    const float mg = s.x / a.hidden, mgx = s.y / a.hidden;
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x)
        dx[i] = from_float<T>(rstd * (to_float(dy[i]) * to_float(w[i]) - mg - (to_float(x[i]) - mean) * rstd * mgx));
}

// one thread per column and slice of rows: partial sums [slices][2][hidden]
template <class T>
__global__ void __launch_bounds__(kNormThreads) layer_norm_columns_kernel(const LayerNormArgs a) {
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= a.hidden) return;
    const int64_t r0 = static_cast<int64_t>(a.rows) * blockIdx.y / gridDim.y, r1 = static_cast<int64_t>(a.rows) * (blockIdx.y + 1) / gridDim.y;
    float dw = 0.f, db = 0.f;
    for (int64_t r = r0; r < r1; ++r) {
        const float d = to_float(reinterpret_cast<const T*>(a.dy)[r * a.lddy + i]);
        dw += d * ((to_float(reinterpret_cast<const T*>(a.x)[r * a.ldx + i]) - a.mean[r]) * a.rstd[r]);
        db += d;
    }
    a.partial[(2ll * blockIdx.y) * a.hidden + i] = dw;
    a.partial[(2ll * blockIdx.y + 1) * a.hidden + i] = db;
}

template <class P>
__global__ void __launch_bounds__(kNormThreads) layer_norm_reduce_kernel(const LayerNormArgs a) {
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= a.hidden) return;
    float dw = 0.f, db = 0.f;
    for (int s = 0; s < a.slices; ++s) {
        dw += a.partial[(2ll * s) * a.hidden + i];
        db += a.partial[(2ll * s + 1) * a.hidden + i];
    }
    reinterpret_cast<P*>(a.dw)[i] = from_float<P>(dw);
    if (a.db != nullptr) reinterpret_cast<P*>(a.db)[i] = from_float<P>(db);
}

template <class F>
cudaError_t launch(F fn, dim3 grid, const LayerNormArgs& a, cudaStream_t stream) {
    void* params[] = {const_cast<LayerNormArgs*>(&a)};
    return launch_dependent(reinterpret_cast<const void*>(fn), grid, dim3(kNormThreads), params, 0, stream);
}

}  // namespace

int layer_norm_slices(int rows, int hidden, int num_sms) {
    const int blocks = (hidden + kNormThreads - 1) / kNormThreads;
    return std::max(1, std::min((rows + 15) / 16, 8 * num_sms / blocks));
}

cudaError_t launch_layer_norm(const LayerNormArgs& a, cudaStream_t stream) {
    if (a.hidden < 1 || a.rows < 0) return cudaErrorInvalidValue;
    if (a.rows == 0) return cudaSuccess;
    const dim3 grid(a.rows);
    if (a.x_bf16) return a.param_bf16 ? launch(layer_norm_kernel<__nv_bfloat16, __nv_bfloat16>, grid, a, stream) : launch(layer_norm_kernel<__nv_bfloat16, float>, grid, a, stream);
    return a.param_bf16 ? launch(layer_norm_kernel<float, __nv_bfloat16>, grid, a, stream) : launch(layer_norm_kernel<float, float>, grid, a, stream);
}

cudaError_t launch_layer_norm_backward(const LayerNormArgs& a, cudaStream_t stream) {
    if (a.hidden < 1 || a.rows < 0 || a.slices < 1) return cudaErrorInvalidValue;
    cudaError_t err = cudaSuccess;
    if (a.rows > 0) {
        const dim3 grid(a.rows);
        if (a.x_bf16) err = a.param_bf16 ? launch(layer_norm_dx_kernel<__nv_bfloat16, __nv_bfloat16>, grid, a, stream) : launch(layer_norm_dx_kernel<__nv_bfloat16, float>, grid, a, stream);
        else err = a.param_bf16 ? launch(layer_norm_dx_kernel<float, __nv_bfloat16>, grid, a, stream) : launch(layer_norm_dx_kernel<float, float>, grid, a, stream);
        if (err != cudaSuccess) return err;
    }
    const int blocks = (a.hidden + kNormThreads - 1) / kNormThreads;
    const dim3 grid(blocks, a.slices);
    err = a.x_bf16 ? launch(layer_norm_columns_kernel<__nv_bfloat16>, grid, a, stream) : launch(layer_norm_columns_kernel<float>, grid, a, stream);
    if (err != cudaSuccess) return err;
    return a.param_bf16 ? launch(layer_norm_reduce_kernel<__nv_bfloat16>, dim3(blocks), a, stream) : launch(layer_norm_reduce_kernel<float>, dim3(blocks), a, stream);
}

}  // namespace ep
