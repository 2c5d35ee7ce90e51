// Orthogonalises a stack of matrices by Newton-Schulz steps (the update of the Muon optimiser).  Per matrix, with rows <= cols (others are
// transposed on their way in and out):
//
//     X = G / (|G|_F + eps);     per step:  A = X X^T,  B = b A + c A A,  X = a X + B X
//
// The three products of a step run on the tensor cores (tcgen05, fp16 operands, 32-bit sums in tensor memory), one persistent kernel each.  A and
// B are symmetric: only tiles on and above the diagonal are computed, the others are written as their mirror images.
//
// Precision.  A step multiplies small singular values by up to a = 3.44, and with them whatever rounding has put there, so what is rounded
// matters more than how often.  Relative error of five steps, simulated in 64 bits for a matrix of normal numbers / one with 32 strong
// directions / with a single one: operands in bf16 1e-2 / 6e-2 / 0.46; in fp16, with a factor that is a power of two for their range,
// 1.3e-3 / 7e-3 / 6e-2, nearly all of it from rounding the X of a X and the diagonals of A and B, which are far larger than what is around them.
// So X is carried in two halves, hi + lo 2^-11 (22 bits; the products read hi alone), and the diagonals are carried in 32 bits beside matrices
// whose diagonal is zero:  A = O + diag(d),  A A = O O + (d_i + d_j) O + diag(d^2),  B X = (B - diag) X + diag X.  Then 5e-4 / 2e-4 / 4e-4, less than
// the rounding of the result to bf16 (1.7e-3).
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "gemm_sm100.cuh"

namespace ep {

namespace {

constexpr int kTileM = 128, kTileK = 64;                       // one 128-byte row of fp16 per stage
constexpr int kNsThreads = 192;                                // TMA warp, MMA warp, four epilogue warps
constexpr float kUnitX = 4096.f, kUnitLo = 2048.f, kUnitA = 1024.f;      // stored = value * unit; lo: unit of hi * kUnitLo
constexpr int kTransposePitch = 72;                            // bytes of a staged column of 32 fp16 values
constexpr int kEpiWarpBytes = 32 * 128 + 32 * kTransposePitch; // 32 x 32 sums, and the same tile transposed
constexpr uint64_t kNsWaitLimitNs = 4ull * 1000 * 1000 * 1000; // when the caller gives no limit

__host__ __device__ constexpr int ns_stages(int block_n) { return block_n == 256 ? 4 : 5; }
__host__ __device__ constexpr int ns_stage_bytes(int block_n) { return (kTileM + block_n) * 128; }
__host__ __device__ constexpr int ns_smem_bytes(int block_n) { return ns_stages(block_n) * ns_stage_bytes(block_n) + 1024 + 4 * kEpiWarpBytes; }

struct NsSmem {
    uint64_t full[8], empty[8], acc_full[2], acc_empty[2], quiet;
    uint32_t tmem_base;
    int failed;
};

// Bounded wait for an mbarrier phase; when it runs out the device's flag is raised, and the status block of the caller's buffer written.
// code: 1 free stage, 2 free accumulator, 4 full stage, 5 finished accumulator
__device__ __noinline__ void ns_fail(const NsReport& r, int* failed, int code) {
    *failed = code;
    if (atomicCAS(r.error, 0, code) == 0 && r.status != nullptr) {
        volatile uint64_t* st = r.status;
        st[EP_STATUS_PHASE] = EP_PH_GEMM_PIPE;
        st[EP_STATUS_PEER] = static_cast<uint64_t>(-1ll);
        st[EP_STATUS_EXPECTED] = static_cast<uint64_t>(code);
        st[EP_STATUS_OBSERVED] = blockIdx.x;
        st[EP_STATUS_RANK] = static_cast<uint64_t>(r.status_rank);
        __threadfence_system();
        st[EP_STATUS_CODE] = EP_ERR_TIMEOUT;
        __threadfence_system();
    }
}
__device__ __forceinline__ bool ns_wait(uint64_t* bar, uint32_t parity, NsSmem* sm, const NsReport& r, int code) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns(), limit = r.timeout_ns != 0 ? r.timeout_ns : kNsWaitLimitNs;
    uint32_t spins = 0;
    while (!ptx::mbar_try_wait(bar, parity)) {
        if ((++spins & 63u) == 0u) {
            if (*reinterpret_cast<volatile int*>(&sm->failed)) return false;
            if (globaltimer_ns() - t0 > limit) {
                ns_fail(r, &sm->failed, code);
                return false;
            }
        }
    }
    return true;
}

template <int kStages>
struct NsPipe {
    int stage = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void advance() {
        if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
        }
    }
};

struct NsTile {
    int g, m, n;             // matrix, 128-row block, kBlockN-column block
    bool mirror;             // symmetric result: the tile's mirror image lies outside what is computed
};
// Symmetric result: column block j is computed for the row blocks 0 .. (j + 1) * kBlockN / 128 - 1.
template <int kBlockN>
__host__ __device__ __forceinline__ int symmetric_tiles(int rows) {
    constexpr int kRatio = kBlockN / kTileM;
    const int num_m = (rows + kTileM - 1) / kTileM, num_n = (rows + kBlockN - 1) / kBlockN;
    return kRatio * num_n * (num_n - 1) / 2 + (num_m < kRatio * num_n ? num_m : kRatio * num_n);
}
template <int kBlockN, bool kSymmetric>
__device__ __forceinline__ NsTile ns_tile(int item, int per_matrix, int num_m) {
    NsTile t;
    t.g = item / per_matrix;
    const int i = item - t.g * per_matrix;
    if constexpr (kSymmetric) {
        constexpr int kRatio = kBlockN / kTileM;
        int n = static_cast<int>((sqrtf(8.f * i / kRatio + 1.f) - 1.f) * 0.5f);
        while (kRatio * n * (n + 1) / 2 > i) --n;
        while (kRatio * (n + 1) * (n + 2) / 2 <= i) ++n;
        t.n = n;
        t.m = i - kRatio * n * (n + 1) / 2;
        t.mirror = t.m < kRatio * n;
    } else {
        t.n = i / num_m;
        t.m = i - t.n * num_m;
        t.mirror = false;
    }
    return t;
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void unpack_half(const int4& v, float (&f)[8]) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = __half22float2(h[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
    }
}

// kMode 0: O, d = X X^T without its diagonal, and the diagonal.  1: B, coef = b A + c A A without its diagonal, and a + the diagonal.
// 2: X <- coef X + B X.
template <int kMode, int kBlockN>
__global__ void __launch_bounds__(kNsThreads, 1)
ns_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ NsArgs g) {
    extern __shared__ __align__(1024) uint8_t smem[];
    constexpr int kStages = ns_stages(kBlockN), kBytesA = kTileM * 128, kBytesB = kBlockN * 128;
    constexpr bool kSymmetric = kMode != 2;
    constexpr int kTmemColumns = 2 * kBlockN;
    constexpr uint32_t kIdesc = umma::make_instr_desc(kTileM, kBlockN, umma::kFormatF16, false, kMode == 2);
    uint8_t* s_a = smem;
    uint8_t* s_b = smem + kStages * kBytesA;
    NsSmem* sm = reinterpret_cast<NsSmem*>(smem + kStages * (kBytesA + kBytesB));
    uint8_t* s_epi = smem + kStages * (kBytesA + kBytesB) + 1024;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int num_m = (g.rows + kTileM - 1) / kTileM;
    const int per_matrix = kSymmetric ? symmetric_tiles<kBlockN>(g.rows) : num_m * ((g.cols + kBlockN - 1) / kBlockN);
    const int num_items = per_matrix * g.count;
    const int num_k = ((kMode == 0 ? g.cols : g.rows) + kTileK - 1) / kTileK;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            ptx::mbar_init(&sm->full[i], 1);
            ptx::mbar_init(&sm->empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&sm->acc_full[i], 1);
            ptx::mbar_init(&sm->acc_empty[i], 4);
        }
        ptx::mbar_init(&sm->quiet, 1);
        sm->failed = 0;
        ptx::mbar_fence_init();
        umma::prefetch_tensormap(&map_a);
        umma::prefetch_tensormap(&map_b);
    }
    if (warp == 1) {
        umma::tmem_alloc(&sm->tmem_base, kTmemColumns);
        umma::tmem_relinquish();
    }
    umma::fence_before_thread_sync();
    __syncthreads();
    umma::fence_after_thread_sync();
    const uint32_t tmem_base = sm->tmem_base;
    ptx::wait_for_previous_kernel();

    if (warp == 0) {
        if (ptx::elect_one()) {
            NsPipe<kStages> p;
            int loads = 0;
            bool ok = true;
            for (int item = blockIdx.x; item < num_items && ok; item += gridDim.x) {
                const NsTile t = ns_tile<kBlockN, kSymmetric>(item, per_matrix, num_m);
                for (int kb = 0; kb < num_k; ++kb) {
                    ok = ns_wait(&sm->empty[p.stage], p.phase ^ 1, sm, g.report, 1);
                    if (!ok) break;
                    ptx::mbar_arrive_expect_tx(&sm->full[p.stage], kBytesA + kBytesB);
                    umma::tma_load_3d(s_a + p.stage * kBytesA, &map_a, kb * kTileK, t.m * kTileM, t.g, &sm->full[p.stage]);
                    if constexpr (kMode == 2) {
#pragma unroll
                        for (int i = 0; i < kBlockN / 64; ++i)
                            umma::tma_load_3d(s_b + p.stage * kBytesB + i * umma::kMnChunkBytes, &map_b, t.n * kBlockN + i * 64, kb * kTileK, t.g, &sm->full[p.stage]);
                    } else {
                        umma::tma_load_3d(s_b + p.stage * kBytesB, &map_b, kb * kTileK, t.n * kBlockN, t.g, &sm->full[p.stage]);
                    }
                    loads = min(loads + 1, kStages);
                    p.advance();
                }
            }
            ptx::let_next_kernel_start();
            if (!ok) {      // give what is still in flight time to land before the shared memory goes to another CTA
                for (; loads > 0; --loads) {
                    p.phase ^= p.stage == 0;
                    p.stage = p.stage == 0 ? kStages - 1 : p.stage - 1;
                    mbar_drain(&sm->full[p.stage], p.phase, 1000000000ull);
                }
            }
        }
    } else if (warp == 1) {
        if (ptx::elect_one()) {
            NsPipe<kStages> p;
            int acc = 0;
            uint32_t acc_phase = 0;
            bool ok = true;
            for (int item = blockIdx.x; item < num_items && ok; item += gridDim.x) {
                ok = ns_wait(&sm->acc_empty[acc], acc_phase ^ 1, sm, g.report, 2);
                if (!ok) break;
                umma::fence_after_thread_sync();
                for (int kb = 0; kb < num_k; ++kb) {
                    ok = ns_wait(&sm->full[p.stage], p.phase, sm, g.report, 4);
                    if (!ok) break;
                    umma::fence_after_thread_sync();
                    const uint64_t desc_a = umma::make_smem_desc_sw128(s_a + p.stage * kBytesA);
                    const uint64_t desc_b = kMode == 2 ? umma::make_smem_desc_mn_sw128(s_b + p.stage * kBytesB) : umma::make_smem_desc_sw128(s_b + p.stage * kBytesB);
                    constexpr int kStepB = kMode == 2 ? 16 * 128 : 32;       // 16 elements of K
#pragma unroll
                    for (int k = 0; k < kTileK / 16; ++k)
                        umma::mma_ss<false>(tmem_base + acc * kBlockN, umma::advance_desc_k(desc_a, k * 32), umma::advance_desc_k(desc_b, k * kStepB), kIdesc,
                                            kb != 0 || k != 0);
                    umma::mma_commit(&sm->empty[p.stage]);
                    p.advance();
                }
                if (!ok) break;
                umma::mma_commit(&sm->acc_full[acc]);
                acc ^= 1;
                acc_phase ^= acc == 0;
            }
            if (!ok) {      // products still under way end before the tensor memory is given back
                umma::mma_commit(&sm->quiet);
                mbar_drain(&sm->quiet, 0, 1000000000ull);
            }
        }
    } else {
        const int quad = warp & 3;
        uint8_t* s_sum = s_epi + quad * kEpiWarpBytes;
        uint8_t* s_t = s_sum + 32 * 128;
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int item = blockIdx.x; item < num_items; item += gridDim.x) {
            const NsTile t = ns_tile<kBlockN, kSymmetric>(item, per_matrix, num_m);
            const bool ok = ns_wait(&sm->acc_full[acc], acc_phase, sm, g.report, 5);
            if (!__all_sync(0xffffffffu, ok)) break;
            umma::fence_after_thread_sync();
            const int row0 = t.m * kTileM + quad * 32;
            const int64_t sq = static_cast<int64_t>(t.g) * g.rows * g.ld_sq, wide = static_cast<int64_t>(t.g) * g.rows * g.ld_x, diag = static_cast<int64_t>(t.g) * g.rows;
            const int width = kSymmetric ? g.ld_sq : g.ld_x;
#pragma unroll 1
            for (int c = 0; c < kBlockN / 32; ++c) {
                const int col0 = t.n * kBlockN + c * 32;
                if (col0 >= width || row0 >= g.rows) break;
                uint32_t r[32];
                umma::tmem_ld_32x32(tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + acc * kBlockN + c * 32, r);
                umma::tmem_ld_wait();
                // one row per lane -> four lanes with eight columns each per row
#pragma unroll
                for (int v = 0; v < 8; ++v)
                    *reinterpret_cast<uint4*>(s_sum + lane * 128 + ((v ^ (lane & 7)) * 16)) = make_uint4(r[4 * v], r[4 * v + 1], r[4 * v + 2], r[4 * v + 3]);
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int lr = i * 8 + (lane >> 2), lc = (lane & 3) * 8, row = row0 + lr, col = col0 + lc;
                    const float4 s0 = *reinterpret_cast<const float4*>(s_sum + lr * 128 + ((((lc >> 2)) ^ (lr & 7)) * 16));
                    const float4 s1 = *reinterpret_cast<const float4*>(s_sum + lr * 128 + ((((lc >> 2) + 1) ^ (lr & 7)) * 16));
                    float v[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
                    const bool in = row < g.rows && col < width;
                    int4 out = make_int4(0, 0, 0, 0);
                    uint32_t* o = reinterpret_cast<uint32_t*>(&out);
                    if constexpr (kMode == 0) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            if (in && row == col + j) {
                                g.diag[diag + row] = v[j] * (1.f / (kUnitX * kUnitX));
                                v[j] = 0.f;
                            }
                            v[j] *= kUnitA / (kUnitX * kUnitX);
                        }
                    } else if constexpr (kMode == 1) {
                        if (in) {
                            float old[8];
                            unpack_half(*reinterpret_cast<const int4*>(g.sq_in + sq + static_cast<int64_t>(row) * g.ld_sq + col), old);
                            const float di = g.diag[diag + row];
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const float dj = col + j < g.rows ? g.diag[diag + col + j] : 0.f;
                                // (B in kUnitA; O O in kUnitA^2)
                                if (row == col + j) {
                                    g.coef[diag + row] = g.a + g.b * di + g.c * (di * di + v[j] * (1.f / (kUnitA * kUnitA)));
                                    v[j] = 0.f;
                                } else {
                                    v[j] = (g.b + g.c * (di + dj)) * old[j] + g.c * (1.f / kUnitA) * v[j];
                                }
                            }
                        }
                    } else {
                        if (in) {
                            const int64_t at = wide + static_cast<int64_t>(row) * g.ld_x + col;
                            float hi[8], lo[8];
                            unpack_half(*reinterpret_cast<const int4*>(g.x_in + at), hi);
                            unpack_half(*reinterpret_cast<const int4*>(g.x_lo + at), lo);
                            const float k = g.coef[diag + row];
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[j] = k * (hi[j] + lo[j] * (1.f / kUnitLo)) + v[j] * (1.f / kUnitA);     // in kUnitX
                        }
                    }
                    if (kMode != 2 || g.out == nullptr) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[j] = pack_half(v[2 * j], v[2 * j + 1]);
                        if (in) *reinterpret_cast<int4*>(kMode == 2 ? g.x_out + wide + static_cast<int64_t>(row) * g.ld_x + col
                                                                     : g.sq_out + sq + static_cast<int64_t>(row) * g.ld_sq + col) = out;
                        if (kMode == 2 && in) {
                            float hi[8];
                            unpack_half(out, hi);
#pragma unroll
                            for (int j = 0; j < 4; ++j) o[j] = pack_half((v[2 * j] - hi[2 * j]) * kUnitLo, (v[2 * j + 1] - hi[2 * j + 1]) * kUnitLo);
                            *reinterpret_cast<int4*>(g.x_lo + wide + static_cast<int64_t>(row) * g.ld_x + col) = out;
                        }
                    } else {
                        // the last step: the result, in the caller's orientation
                        __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(g.out) + static_cast<int64_t>(t.g) * g.rows * g.cols;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j] * (1.f / kUnitX), v[2 * j + 1] * (1.f / kUnitX));
                            o[j] = *reinterpret_cast<const uint32_t*>(&h);
                        }
                        if (in && !g.out_transposed) {
                            dst += static_cast<int64_t>(row) * g.cols + col;
                            if (g.cols % 8 == 0) {
                                *reinterpret_cast<int4*>(dst) = out;
                            } else {
#pragma unroll
                                for (int j = 0; j < 8; ++j)
                                    if (col + j < g.cols) reinterpret_cast<uint16_t*>(dst)[j] = static_cast<uint16_t>(o[j >> 1] >> (16 * (j & 1)));
                            }
                        }
                    }
                    if (t.mirror || (kMode == 2 && g.out != nullptr && g.out_transposed)) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            *reinterpret_cast<uint16_t*>(s_t + (lc + j) * kTransposePitch + lr * 2) = static_cast<uint16_t>(o[j >> 1] >> (16 * (j & 1)));
                    }
                }
                __syncwarp();
                if (t.mirror || (kMode == 2 && g.out != nullptr && g.out_transposed)) {
                    // rows of the mirror image: 32 values, eight lanes with four each
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int lr = i * 4 + (lane >> 3), lc = (lane & 7) * 4, row = col0 + lr, col = row0 + lc;
                        const uint2 v = *reinterpret_cast<const uint2*>(s_t + lr * kTransposePitch + lc * 2);
                        if constexpr (kMode != 2) {
                            if (row < g.rows && col < g.ld_sq) *reinterpret_cast<uint2*>(g.sq_out + sq + static_cast<int64_t>(row) * g.ld_sq + col) = v;
                        } else {
                            uint16_t* dst = reinterpret_cast<uint16_t*>(g.out) + static_cast<int64_t>(t.g) * g.rows * g.cols + static_cast<int64_t>(row) * g.rows + col;
                            if (row < g.cols) {
                                if (g.rows % 4 == 0) {
                                    if (col < g.rows) *reinterpret_cast<uint2*>(dst) = v;
                                } else {
#pragma unroll
                                    for (int j = 0; j < 4; ++j)
                                        if (col + j < g.rows) dst[j] = static_cast<uint16_t>((j < 2 ? v.x : v.y) >> (16 * (j & 1)));
                                }
                            }
                        }
                    }
                    __syncwarp();
                }
            }
            umma::fence_before_thread_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&sm->acc_empty[acc]);
            acc ^= 1;
            acc_phase ^= acc == 0;
        }
    }
    umma::fence_before_thread_sync();
    __syncthreads();
    if (warp == 1) umma::tmem_dealloc(tmem_base, kTmemColumns);
}

// ------------------------------------------------------------------------------------------------ the first X
constexpr int kNormThreads = 256, kCastTile = 64;

template <class T>
__device__ __forceinline__ float as_float(T v) {
    if constexpr (sizeof(T) == 2) return __bfloat162float(v);
    else return v;
}

// sums of squares, in 64 bits: one per CTA
template <class T>
__global__ void __launch_bounds__(kNormThreads) ns_norm_kernel(const NsArgs g) {
    __shared__ double s_sum[kNormThreads / 32];
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const T* src = reinterpret_cast<const T*>(g.in) + static_cast<int64_t>(blockIdx.y) * g.in_stride_matrix;
    double sum = 0.0;
    for (int64_t line = blockIdx.x; line < g.in_lines; line += gridDim.x) {
        const T* p = src + line * g.in_stride_line;
        for (int i = threadIdx.x; i < g.in_line; i += kNormThreads) {
            const double v = as_float(p[i]);
            sum += v * v;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kNormThreads / 32; ++w) sum += s_sum[w];
        g.norm_parts[static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x] = sum;
    }
}

// X = G / (norm + eps) as hi + lo, with rows <= cols; lines of the input are rows of X, or (flip) its columns.  One CTA per 64 x 64 tile.
template <class T>
__global__ void __launch_bounds__(kNormThreads) ns_cast_kernel(const NsArgs g) {
    __shared__ float tile[kCastTile][kCastTile + 1];
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const int line0 = blockIdx.y * kCastTile, at0 = blockIdx.x * kCastTile;
    const T* src = reinterpret_cast<const T*>(g.in) + static_cast<int64_t>(blockIdx.z) * g.in_stride_matrix;
    double sum = 0.0;
    for (int i = 0; i < g.num_norm_parts; ++i) sum += g.norm_parts[static_cast<int64_t>(blockIdx.z) * g.num_norm_parts + i];
    const double scale = static_cast<double>(kUnitX) / (sqrt(sum) + static_cast<double>(g.eps));
    for (int i = threadIdx.x; i < kCastTile * kCastTile; i += kNormThreads) {
        const int l = i / kCastTile, c = i % kCastTile;
        const float v = line0 + l < g.in_lines && at0 + c < g.in_line ? static_cast<float>(as_float(src[(line0 + l) * g.in_stride_line + at0 + c]) * scale) : 0.f;
        if (g.flip) tile[c][l] = v;
        else tile[l][c] = v;
    }
    __syncthreads();
    const int row0 = g.flip ? at0 : line0, col0 = g.flip ? line0 : at0;
    for (int i = threadIdx.x; i < kCastTile * kCastTile; i += kNormThreads) {
        const int r = i / kCastTile, c = i % kCastTile;
        if (row0 + r < g.rows && col0 + c < g.ld_x) {
            const int64_t at = (static_cast<int64_t>(blockIdx.z) * g.rows + row0 + r) * g.ld_x + col0 + c;
            const __half hi = __float2half_rn(tile[r][c]);
            g.x_out[at] = hi;
            g.x_lo[at] = __float2half_rn((tile[r][c] - __half2float(hi)) * kUnitLo);
        }
    }
}

bool make_map(CUtensorMap* map, const __half* base, int64_t count, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
    EncodeTiledFn encode = get_encode_fn();
    if (encode == nullptr) return false;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(count)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld * 2), static_cast<cuuint64_t>(rows * ld * 2)};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_rows), 1};
    const cuuint32_t elem_strides[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(base), dims, strides, box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int kMode, int kBlockN>
cudaError_t launch_product(const CUtensorMap& map_a, const CUtensorMap& map_b, const NsArgs& g, int num_sms, cudaStream_t stream) {
    const void* fn = reinterpret_cast<const void*>(ns_kernel<kMode, kBlockN>);
    const cudaError_t err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, ns_smem_bytes(kBlockN));
    if (err != cudaSuccess) return err;
    const int64_t num_m = (g.rows + kTileM - 1) / kTileM;
    const int64_t items = g.count * (kMode != 2 ? static_cast<int64_t>(symmetric_tiles<kBlockN>(g.rows)) : num_m * ((g.cols + kBlockN - 1) / kBlockN));
    void* params[] = {const_cast<CUtensorMap*>(&map_a), const_cast<CUtensorMap*>(&map_b), const_cast<NsArgs*>(&g)};
    return launch_dependent(fn, dim3(static_cast<unsigned>(std::min<int64_t>(items, num_sms))), dim3(kNsThreads), params, ns_smem_bytes(kBlockN), stream);
}

int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }

}  // namespace

// Workspace: hi of X twice and lo once, O and B, their diagonals, sums of squares.
NsWorkspace newton_schulz_workspace(int64_t count, int64_t rows, int64_t cols, int num_sms) {
    NsWorkspace w{};
    w.ld_x = round8(cols);
    w.ld_sq = round8(rows);
    w.norm_parts = std::max<int64_t>(1, std::min<int64_t>(rows, 4 * num_sms / std::max<int64_t>(1, count)));
    auto take = [&](int64_t bytes) {
        const int64_t at = w.bytes;
        w.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    w.norms = take(count * w.norm_parts * 8);
    for (int64_t& x : w.x) x = take(count * rows * w.ld_x * 2);
    w.lo = take(count * rows * w.ld_x * 2);
    for (int64_t& s : w.sq) s = take(count * rows * w.ld_sq * 2);
    for (int64_t& d : w.diag) d = take(count * rows * 4);
    return w;
}

cudaError_t launch_newton_schulz(const NsArgs& args, const NsWorkspace& w, uint8_t* workspace, int steps, int num_sms, cudaStream_t stream) {
    if (args.count < 1 || args.rows < 1 || args.rows > args.cols || steps < 1 || reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return cudaErrorInvalidValue;
    NsArgs g = args;
    g.ld_x = static_cast<int>(w.ld_x);
    g.ld_sq = static_cast<int>(w.ld_sq);
    __half *x[2], *sq[2];
    for (int i = 0; i < 2; ++i) {
        x[i] = reinterpret_cast<__half*>(workspace + w.x[i]);
        sq[i] = reinterpret_cast<__half*>(workspace + w.sq[i]);
    }
    g.x_lo = reinterpret_cast<__half*>(workspace + w.lo);
    g.diag = reinterpret_cast<float*>(workspace + w.diag[0]);
    g.coef = reinterpret_cast<float*>(workspace + w.diag[1]);
    g.norm_parts = reinterpret_cast<double*>(workspace + w.norms);
    g.num_norm_parts = static_cast<int>(w.norm_parts);
    void* out = g.out;
    g.out = nullptr;
    constexpr int kBlockN = 256;
    CUtensorMap x_rows[2], x_cols[2], x_mn[2], o_rows, o_cols, b_rows;
    for (int i = 0; i < 2; ++i)
        if (!make_map(&x_rows[i], x[i], g.count, g.rows, g.cols, g.ld_x, kTileM) || !make_map(&x_cols[i], x[i], g.count, g.rows, g.cols, g.ld_x, kBlockN) ||
            !make_map(&x_mn[i], x[i], g.count, g.rows, g.cols, g.ld_x, 64))
            return cudaErrorInvalidValue;
    if (!make_map(&o_rows, sq[0], g.count, g.rows, g.rows, g.ld_sq, kTileM) || !make_map(&o_cols, sq[0], g.count, g.rows, g.rows, g.ld_sq, kBlockN) ||
        !make_map(&b_rows, sq[1], g.count, g.rows, g.rows, g.ld_sq, kTileM))
        return cudaErrorInvalidValue;

    void* params[] = {&g};
    g.x_out = x[0];
    const dim3 norm_grid(g.num_norm_parts, g.count);
    const dim3 cast_grid((g.in_line + kCastTile - 1) / kCastTile, static_cast<unsigned>((g.in_lines + kCastTile - 1) / kCastTile), g.count);
    cudaError_t err = launch_dependent(g.in_bf16 ? reinterpret_cast<const void*>(ns_norm_kernel<__nv_bfloat16>) : reinterpret_cast<const void*>(ns_norm_kernel<float>), norm_grid,
                                       dim3(kNormThreads), params, 0, stream);
    if (err != cudaSuccess) return err;
    err = launch_dependent(g.in_bf16 ? reinterpret_cast<const void*>(ns_cast_kernel<__nv_bfloat16>) : reinterpret_cast<const void*>(ns_cast_kernel<float>), cast_grid,
                           dim3(kNormThreads), params, 0, stream);
    for (int s = 0; s < steps && err == cudaSuccess; ++s) {
        const int from = s & 1;
        g.sq_out = sq[0];
        err = launch_product<0, kBlockN>(x_rows[from], x_cols[from], g, num_sms, stream);
        if (err != cudaSuccess) break;
        g.sq_in = sq[0];
        g.sq_out = sq[1];
        err = launch_product<1, kBlockN>(o_rows, o_cols, g, num_sms, stream);
        if (err != cudaSuccess) break;
        g.x_in = x[from];
        g.x_out = x[from ^ 1];
        if (s == steps - 1) g.out = out;
        err = launch_product<2, kBlockN>(b_rows, x_mn[from], g, num_sms, stream);
    }
    return err;
}

}  // namespace ep
