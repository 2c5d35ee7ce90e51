// Orthogonalises a stack of matrices by Newton-Schulz steps (the update of the Muon optimiser).  Per matrix, with rows <= cols (others are
// transposed on their way in and out):
//
//     X = G / (|G|_F + eps);     per step:  A = X X^T,  B = b A + c A A,  X = a X + B X
//
// The first two steps may go as a pair, without the X between them. With Q = a I + B the next A is Q A Q, so that a pair is
//
//     A = X X^T,  Q1 = a I + b A + c A A,  T = Q1 A,  A = T Q1,  Q2 = a I + b A + c A A,  Q = Q2 Q1,  X = Q X
//
// where all but the first and the last are symmetric products of rows^3, computed by half: in multiply-adds 3 cols/rows + 5 halves of 2 rows^3 for
// the pair, 6 cols/rows + 2 for two single steps.
//
// The products run on the tensor cores (tcgen05, fp16 operands, 32-bit sums in tensor memory), one persistent kernel each.  A and
// B are symmetric: only tiles on and above the diagonal are computed, the others are written as their mirror images.
//
// Precision.  A step multiplies small singular values by up to a = 3.44, and with them whatever rounding has put there, so what is rounded
// matters more than how often.  Relative error of five steps, simulated in 64 bits for a matrix of normal numbers / one with 32 strong
// directions / with a single one: operands in bf16 1e-2 / 6e-2 / 0.46; in fp16, with a factor that is a power of two for their range,
// 1.3e-3 / 7e-3 / 6e-2, nearly all of it from rounding the X of a X and the diagonals of A and B, which are far larger than what is around them.
// So X is carried in two halves, hi + lo 2^-11 (22 bits; the products read hi alone), and the diagonals are carried in 32 bits beside matrices
// whose diagonal is zero:  A = O + diag(d),  A A = O O + (d_i + d_j) O + diag(d^2),  B X = (B - diag) X + diag X.  Then 5e-4 / 2e-4 / 4e-4, less than
// the rounding of the result to bf16 (1.7e-3).  Singular
// values on two levels far apart take the most: 1.9e-3 for 512 rows (a fifth of them at one, the others at a thousandth), 2.9e-3 for 256, 3.9e-3, 5e-3, 8e-3 and 2e-2 for 128, 64, 32 and 16,
// where fewer roundings average out.  In a pair the second A comes from the first, not from X, and what its small eigenvalues are off by
// has been multiplied by a^2.  The steps after a first pair, each from its own X, make that good: the same errors as single steps for 47 spectra at 512
// and 1024 rows.  A second pair would not: 6.8e-3, four times the rounding of the result, for a tenth of 512 singular values at one and the others at 0.1, where single steps give 6e-4.  At
// 64 rows a pair is off by 1.9e-3 for normal numbers; three steps at once are off by 2e-3 with a single strong direction, five are no number at all: so a pair, and only from 512 rows.
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "common.cuh"
#include "gemm_sm100.cuh"

namespace ep {

namespace {

constexpr int kTileM = 128, kTileK = 64;                       // one 128-byte row of fp16 per stage
constexpr int kEpiWarps = 8, kNsThreads = 64 + kEpiWarps * 32; // TMA warp, MMA warp, eight epilogue warps (two per 32 tile rows, half of the columns each)
constexpr float kUnitX = 4096.f, kUnitLo = 2048.f, kUnitA = 1024.f;      // stored = value * unit; lo: unit of hi * kUnitLo
constexpr int kStagingBytes = 32 * 128;                        // per epilogue warp: 32 x 32 sums, later the same values in fp16 transposed
constexpr int kTransposePitch = 72;                            // bytes of a staged column of 32 fp16 values
constexpr uint64_t kNsWaitLimitNs = 4ull * 1000 * 1000 * 1000; // when the caller gives no limit

__host__ __device__ constexpr int ns_stages(int block_n) { return block_n == 128 ? 6 : 4; }
__host__ __device__ constexpr int ns_tmem_columns(int block_n) { return block_n == 128 ? 256 : 512; }      // two accumulators, a power of two
__host__ __device__ constexpr int ns_stage_bytes(int block_n) { return (kTileM + block_n) * 128; }
__host__ __device__ constexpr int ns_smem_bytes(int block_n) { return ns_stages(block_n) * ns_stage_bytes(block_n) + 1024 + kEpiWarps * kStagingBytes; }

// What a kernel makes of its sums
enum { kGram = 0, kPoly = 1, kUpdate = 2, kGramPart = 3, kProduct = 4 };

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
__device__ __forceinline__ void unpack_half(const uint4& v, float (&f)[8]) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = __half22float2(h[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
    }
}

// 32 x 32 values of a tile lie on a warp as four rows (i * 8 + lane / 4) of eight neighbouring columns ((lane & 3) * 8) per lane: rows are read and written in
// whole sectors.
struct Block {
    int row0, col0;
    __device__ __forceinline__ int row(int i) const { return row0 + i * 8 + ((threadIdx.x & 31) >> 2); }
    __device__ __forceinline__ int col() const { return col0 + (threadIdx.x & 3) * 8; }
    __device__ __forceinline__ bool on_diagonal(int i) const { return static_cast<uint32_t>(row(i) - col()) < 8u; }      // the lane's eight of row i hold it
};
// Value `at` of eight (0 if there is none), which is zero afterwards.  (Looked for by blocks on the diagonal alone: 32 tests per block took ten times as long as all
// else that is done with its values.)
__device__ __forceinline__ float take_diagonal(float (&v)[8], int at) {
    float d = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        d = j == at ? v[j] : d;
        v[j] = j == at ? 0.f : v[j];
    }
    return d;
}
// From one row per lane, as tensor memory gives them
__device__ __forceinline__ void spread(uint8_t* staging, const uint32_t (&r)[32], float (&v)[4][8]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int p = 0; p < 8; ++p)
        *reinterpret_cast<uint4*>(staging + lane * 128 + ((p ^ (lane & 7)) * 16)) = make_uint4(r[4 * p], r[4 * p + 1], r[4 * p + 2], r[4 * p + 3]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int lr = i * 8 + (lane >> 2), p = (lane & 3) * 2;
        const float4 a = *reinterpret_cast<const float4*>(staging + lr * 128 + ((p ^ (lr & 7)) * 16));
        const float4 b = *reinterpret_cast<const float4*>(staging + lr * 128 + (((p + 1) ^ (lr & 7)) * 16));
        v[i][0] = a.x, v[i][1] = a.y, v[i][2] = a.z, v[i][3] = a.w;
        v[i][4] = b.x, v[i][5] = b.y, v[i][6] = b.z, v[i][7] = b.w;
    }
    __syncwarp();
}
// 16-bit values of the block (four words per row) transposed: `write(row, col, four values)` of the mirror image, eight lanes per row of 32
template <class Write>
__device__ __forceinline__ void transposed(uint8_t* staging, const uint32_t (&o)[4][4], const Block& b, Write write) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint16_t*>(staging + ((lane & 3) * 8 + j) * kTransposePitch + (i * 8 + (lane >> 2)) * 2) = static_cast<uint16_t>(o[i][j >> 1] >> (16 * (j & 1)));
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int lr = i * 4 + (lane >> 3), lc = (lane & 7) * 4;
        write(b.col0 + lr, b.row0 + lc, *reinterpret_cast<const uint2*>(staging + lr * kTransposePitch + lc * 2));
    }
    __syncwarp();
}
// The block as it is (or transposed: `o` staged so) row by row, a lane per value: for results whose rows do not start on 16 bytes, where eight lanes' pieces of
// two bytes each took twice the time of the whole product.
template <class Write>
__device__ __forceinline__ void by_value(uint8_t* staging, const uint32_t (&o)[4][4], const Block& b, bool transpose, Write write) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = i * 8 + (lane >> 2), c = (lane & 3) * 8 + j;
            *reinterpret_cast<uint16_t*>(staging + (transpose ? c * kTransposePitch + r * 2 : r * kTransposePitch + c * 2)) = static_cast<uint16_t>(o[i][j >> 1] >> (16 * (j & 1)));
        }
    __syncwarp();
#pragma unroll 8
    for (int r = 0; r < 32; ++r)
        write((transpose ? b.col0 : b.row0) + r, (transpose ? b.row0 : b.col0) + lane, *reinterpret_cast<const uint16_t*>(staging + r * kTransposePitch + lane * 2));
    __syncwarp();
}
// A symmetric result's block, and its mirror image
__device__ __forceinline__ void store_symmetric(const NsArgs& g, uint8_t* staging, int matrix, const Block& b, const float (&v)[4][8], bool mirror) {
    __half* out = g.sq_out + static_cast<int64_t>(matrix) * g.rows * g.ld_sq;
    uint32_t o[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = pack_half(v[i][2 * j], v[i][2 * j + 1]);
        if (b.row(i) < g.rows && b.col() < g.ld_sq)
            *reinterpret_cast<uint4*>(out + static_cast<int64_t>(b.row(i)) * g.ld_sq + b.col()) = make_uint4(o[i][0], o[i][1], o[i][2], o[i][3]);
    }
    if (mirror)
        transposed(staging, o, b, [&](int row, int col, const uint2& four) {
            if (row < g.rows && col < g.ld_sq) *reinterpret_cast<uint2*>(out + static_cast<int64_t>(row) * g.ld_sq + col) = four;
        });
}
// X X^T in kUnitX^2 -> O and the diagonal.  (Columns past the end are sums of zeros.)
__device__ __forceinline__ void finish_gram(const NsArgs& g, uint8_t* staging, int matrix, const Block& b, float (&v)[4][8], bool mirror) {
    if (b.row0 == b.col0)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float d = take_diagonal(v[i], b.row(i) - b.col());
            if (b.on_diagonal(i) && b.row(i) < g.rows) g.diag_out[static_cast<int64_t>(matrix) * g.ld_sq + b.row(i)] = d * (1.f / (kUnitX * kUnitX));
        }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= kUnitA / (kUnitX * kUnitX);
    store_symmetric(g, staging, matrix, b, v, mirror);
}

// B X in kUnitA kUnitX, the old X and the diagonal of Q -> the new X, or (the last step) the result
__device__ __forceinline__ void finish_update(const NsArgs& g, uint8_t* staging, int matrix, const Block& b, float (&v)[4][8], const uint4 (&old)[4], const uint4 (&low)[4],
                                              const float (&row_value)[4]) {
    const int64_t wide = static_cast<int64_t>(matrix) * g.rows * g.ld_x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float hi[8], lo[8];
        unpack_half(old[i], hi);
        unpack_half(low[i], lo);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = row_value[i] * (hi[j] + lo[j] * (1.f / kUnitLo)) + v[i][j] * (1.f / kUnitA);     // in kUnitX
    }
    if (g.out == nullptr) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t o[4], l[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[j] = pack_half(v[i][2 * j], v[i][2 * j + 1]);
                const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&o[j]));
                l[j] = pack_half((v[i][2 * j] - hi.x) * kUnitLo, (v[i][2 * j + 1] - hi.y) * kUnitLo);
            }
            if (b.row(i) < g.rows && b.col() < g.ld_x) {
                const int64_t at = wide + static_cast<int64_t>(b.row(i)) * g.ld_x + b.col();
                *reinterpret_cast<uint4*>(g.x_out + at) = make_uint4(o[0], o[1], o[2], o[3]);
                *reinterpret_cast<uint4*>(g.x_lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
            }
        }
    } else {
        // the last step: the result, in the caller's orientation
        uint16_t* dst = reinterpret_cast<uint16_t*>(g.out) + static_cast<int64_t>(matrix) * g.rows * g.cols;
        uint32_t o[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[i][2 * j] * (1.f / kUnitX), v[i][2 * j + 1] * (1.f / kUnitX));
                o[i][j] = *reinterpret_cast<const uint32_t*>(&h);
            }
        const int out_rows = g.out_transposed ? g.cols : g.rows, out_cols = g.out_transposed ? g.rows : g.cols;
        if (out_cols % 8 != 0) {
            by_value(staging, o, b, g.out_transposed != 0, [&](int row, int col, uint16_t value) {
                if (row < out_rows && col < out_cols) dst[static_cast<int64_t>(row) * out_cols + col] = value;
            });
        } else if (g.out_transposed) {
            transposed(staging, o, b, [&](int row, int col, const uint2& four) {
                if (row < out_rows && col < out_cols) *reinterpret_cast<uint2*>(dst + static_cast<int64_t>(row) * out_cols + col) = four;
            });
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (b.row(i) < out_rows && b.col() < out_cols)
                    *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(b.row(i)) * out_cols + b.col()) = make_uint4(o[i][0], o[i][1], o[i][2], o[i][3]);
        }
    }
}

// What a product of `mode` runs over
template <int kMode, int kBlockN>
struct NsWork {
    static constexpr bool kSymmetric = kMode != kUpdate;
    int num_m, per_matrix, num_tiles, num_items, num_k, splits;
    __device__ __forceinline__ explicit NsWork(const NsArgs& g) {
        num_m = (g.rows + kTileM - 1) / kTileM;
        per_matrix = kSymmetric ? symmetric_tiles<kBlockN>(g.rows) : num_m * ((g.cols + kBlockN - 1) / kBlockN);
        splits = kMode == kGramPart ? g.k_splits : 1;
        num_tiles = per_matrix * g.count;
        num_items = num_tiles * splits;
        num_k = ((kMode == kGram || kMode == kGramPart ? g.cols : g.rows) + kTileK - 1) / kTileK;
    }
    // the K blocks of an item: all, or those of its part
    __device__ __forceinline__ int k_begin(int item) const { return kMode == kGramPart ? num_k * (item / num_tiles) / splits : 0; }
    __device__ __forceinline__ int k_end(int item) const { return kMode == kGramPart ? num_k * (item / num_tiles + 1) / splits : num_k; }
    __device__ __forceinline__ NsTile tile(int item) const { return ns_tile<kBlockN, kSymmetric>(kMode == kGramPart ? item % num_tiles : item, per_matrix, num_m); }
};
template <int kBlockN>
struct NsShared {
    static constexpr int kStages = ns_stages(kBlockN), kBytesA = kTileM * 128, kBytesB = kBlockN * 128;
    uint8_t *a, *b, *staging;
    NsSmem* sm;
    __device__ __forceinline__ explicit NsShared(uint8_t* smem)
        : a(smem), b(smem + kStages * kBytesA), staging(smem + kStages * (kBytesA + kBytesB) + 1024), sm(reinterpret_cast<NsSmem*>(smem + kStages * (kBytesA + kBytesB))) {}
};
template <int kBlockN>
using NsRing = NsPipe<ns_stages(kBlockN)>;

// One thread: requests the operands of this CTA's tiles
template <int kMode, int kBlockN>
__device__ __forceinline__ bool ns_load(const NsArgs& g, const NsShared<kBlockN>& s, const CUtensorMap* map_a, const CUtensorMap* map_b, NsRing<kBlockN>& p, int& loads) {
    const NsWork<kMode, kBlockN> work(g);
    constexpr int kBytesA = NsShared<kBlockN>::kBytesA, kBytesB = NsShared<kBlockN>::kBytesB;
    for (int item = blockIdx.x; item < work.num_items; item += gridDim.x) {
        const NsTile t = work.tile(item);
        const int kb1 = work.k_end(item);
        for (int kb = work.k_begin(item); kb < kb1; ++kb) {
            if (!ns_wait(&s.sm->empty[p.stage], p.phase ^ 1, s.sm, g.report, 1)) return false;
            ptx::mbar_arrive_expect_tx(&s.sm->full[p.stage], kBytesA + kBytesB);
            umma::tma_load_3d(s.a + p.stage * kBytesA, map_a, kb * kTileK, t.m * kTileM, t.g, &s.sm->full[p.stage]);
            if constexpr (kMode == kUpdate) {
#pragma unroll
                for (int i = 0; i < kBlockN / 64; ++i)
                    umma::tma_load_3d(s.b + p.stage * kBytesB + i * umma::kMnChunkBytes, map_b, t.n * kBlockN + i * 64, kb * kTileK, t.g, &s.sm->full[p.stage]);
            } else {
                umma::tma_load_3d(s.b + p.stage * kBytesB, map_b, kb * kTileK, t.n * kBlockN, t.g, &s.sm->full[p.stage]);
            }
            loads = min(loads + 1, NsShared<kBlockN>::kStages);
            p.advance();
        }
    }
    return true;
}
// gives what is still in flight time to land
template <int kBlockN>
__device__ __forceinline__ void ns_drain(const NsShared<kBlockN>& s, NsRing<kBlockN> p, int loads) {
    for (; loads > 0; --loads) {
        p.phase ^= p.stage == 0;
        p.stage = p.stage == 0 ? NsShared<kBlockN>::kStages - 1 : p.stage - 1;
        mbar_drain(&s.sm->full[p.stage], p.phase, 1000000000ull);
    }
}
// One thread: issues the products
template <int kMode, int kBlockN>
__device__ __forceinline__ bool ns_multiply(const NsArgs& g, const NsShared<kBlockN>& s, uint32_t tmem_base, NsRing<kBlockN>& p, int& acc, uint32_t& acc_phase) {
    const NsWork<kMode, kBlockN> work(g);
    constexpr uint32_t kIdesc = umma::make_instr_desc(kTileM, kBlockN, umma::kFormatF16, false, kMode == kUpdate);
    constexpr int kBytesA = NsShared<kBlockN>::kBytesA, kBytesB = NsShared<kBlockN>::kBytesB;
    for (int item = blockIdx.x; item < work.num_items; item += gridDim.x) {
        if (!ns_wait(&s.sm->acc_empty[acc], acc_phase ^ 1, s.sm, g.report, 2)) return false;
        umma::fence_after_thread_sync();
        const int kb0 = work.k_begin(item), kb1 = work.k_end(item);
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!ns_wait(&s.sm->full[p.stage], p.phase, s.sm, g.report, 4)) return false;
            umma::fence_after_thread_sync();
            const uint64_t desc_a = umma::make_smem_desc_sw128(s.a + p.stage * kBytesA);
            const uint64_t desc_b = kMode == kUpdate ? umma::make_smem_desc_mn_sw128(s.b + p.stage * kBytesB) : umma::make_smem_desc_sw128(s.b + p.stage * kBytesB);
            constexpr int kStepB = kMode == kUpdate ? 16 * 128 : 32;       // 16 elements of K
#pragma unroll
            for (int k = 0; k < kTileK / 16; ++k)
                umma::mma_ss<false>(tmem_base + acc * kBlockN, umma::advance_desc_k(desc_a, k * 32), umma::advance_desc_k(desc_b, k * kStepB), kIdesc, kb != kb0 || k != 0);
            umma::mma_commit(&s.sm->empty[p.stage]);
            p.advance();
        }
        umma::mma_commit(&s.sm->acc_full[acc]);
        acc ^= 1;
        acc_phase ^= acc == 0;
    }
    return true;
}
// Eight warps: kGram: O, d = X X^T without its diagonal, and the diagonal; kGramPart: its sums over a part of K.  kPoly: B, coef = b A + c A A without its diagonal, and
// a + the diagonal.  kProduct: P R of two symmetric matrices that commute, likewise.  kUpdate: X <- Q X.
template <int kMode, int kBlockN>
__device__ __forceinline__ bool ns_finish(const NsArgs& g, const NsShared<kBlockN>& s, uint32_t tmem_base, int& acc, uint32_t& acc_phase) {
    const NsWork<kMode, kBlockN> work(g);
    constexpr int kChunks = kBlockN / 2 / 32;          // 32-column blocks of a warp
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = warp & 3, half = (warp - 2) >> 2;
    uint8_t* staging = s.staging + (warp - 2) * kStagingBytes;
    for (int item = blockIdx.x; item < work.num_items; item += gridDim.x) {
        const NsTile t = work.tile(item);
        const int64_t sq = static_cast<int64_t>(t.g) * g.rows * g.ld_sq, wide = static_cast<int64_t>(t.g) * g.rows * g.ld_x, diag = static_cast<int64_t>(t.g) * g.ld_sq;
        const int width = kMode != kUpdate ? g.ld_sq : g.ld_x;
        auto block = [&](int c) { return Block{t.m * kTileM + quad * 32, t.n * kBlockN + half * (kBlockN / 2) + c * 32}; };
        auto empty = [&](const Block& b) { return b.row0 >= g.rows || b.col0 >= width; };
        // What the sums are combined with is requested a block ahead, that of the first one before the sums are there: waiting for it block by block
        // took ten times as long as the products of a tile of 256 K.
        uint4 old[2][4], low[2][4];
        float row_value[4], col_value[2][8];
        auto request = [&](int c, uint4 (&o)[4], uint4 (&l)[4], float (&cv)[8]) {
            const Block b = block(c);
            if (empty(b)) return;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = b.row(i) < g.rows && b.col() < width;
                o[i] = l[i] = make_uint4(0, 0, 0, 0);
                if constexpr (kMode == kPoly || kMode == kProduct) {
                    if (in) {
                        const int64_t at = sq + static_cast<int64_t>(b.row(i)) * g.ld_sq + b.col();
                        o[i] = *reinterpret_cast<const uint4*>(g.sq_in + at);
                        if constexpr (kMode == kProduct) l[i] = *reinterpret_cast<const uint4*>(g.sq_in2 + at);
                    }
                } else if constexpr (kMode == kUpdate) {
                    if (in) {
                        const int64_t at = wide + static_cast<int64_t>(b.row(i)) * g.ld_x + b.col();
                        o[i] = *reinterpret_cast<const uint4*>(g.x_in + at);
                        l[i] = *reinterpret_cast<const uint4*>(g.x_lo + at);
                    }
                }
            }
            if constexpr (kMode == kPoly || kMode == kProduct) {
                const float* values = kMode == kPoly ? g.diag_in : g.diag_in2;
#pragma unroll
                for (int j = 0; j < 8; ++j) cv[j] = b.col() + j < g.rows ? values[diag + b.col() + j] : 0.f;
            }
        };
        if constexpr (kMode == kPoly || kMode == kUpdate || kMode == kProduct) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = block(0).row(i);
                row_value[i] = row >= g.rows ? 0.f : g.diag_in[diag + row];
            }
            request(0, old[0], low[0], col_value[0]);
        }
        const bool ok = ns_wait(&s.sm->acc_full[acc], acc_phase, s.sm, g.report, 5);
        if (!__all_sync(0xffffffffu, ok)) return false;
        umma::fence_after_thread_sync();
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const Block b = block(c);
            if (kMode != kGramPart && empty(b)) break;
            if constexpr (kMode == kPoly || kMode == kUpdate || kMode == kProduct)
                if (c + 1 < kChunks) request(c + 1, old[(c + 1) & 1], low[(c + 1) & 1], col_value[(c + 1) & 1]);
            float v[4][8];
            {
                uint32_t r[32];
                umma::tmem_ld_32x32(tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + acc * kBlockN + half * (kBlockN / 2) + c * 32, r);
                umma::tmem_ld_wait();
                spread(staging, r, v);
            }
            if constexpr (kMode == kGram) {
                finish_gram(g, staging, t.g, b, v, t.mirror);
            } else if constexpr (kMode == kGramPart) {
                // [part][tile][128][kBlockN]
                float* part = g.parts + static_cast<int64_t>(item) * kTileM * kBlockN + (b.col0 - t.n * kBlockN + (lane & 3) * 8);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float* p = part + (b.row(i) - t.m * kTileM) * kBlockN;
                    *reinterpret_cast<float4*>(p) = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
                    *reinterpret_cast<float4*>(p + 4) = make_float4(v[i][4], v[i][5], v[i][6], v[i][7]);
                }
            } else if constexpr (kMode == kPoly) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float f[8];
                    unpack_half(old[c & 1][i], f);
                    const float di = row_value[i], coefficient = g.b + g.c * di;
                    if (b.row0 == b.col0) {
                        const float d = take_diagonal(v[i], b.row(i) - b.col());
                        if (b.on_diagonal(i) && b.row(i) < g.rows) g.diag_out[diag + b.row(i)] = g.a + g.b * di + g.c * (di * di + d * (1.f / (kUnitA * kUnitA)));
                    }
                    // (B in kUnitA; O O in kUnitA^2; O is zero on the diagonal)
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[i][j] = (coefficient + g.c * col_value[c & 1][j]) * f[j] + g.c * (1.f / kUnitA) * v[i][j];
                }
                store_symmetric(g, staging, t.g, b, v, t.mirror);
            } else if constexpr (kMode == kProduct) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float f[8], h[8];
                    unpack_half(old[c & 1][i], f);
                    unpack_half(low[c & 1][i], h);
                    if (b.row0 == b.col0) {
                        const float d = take_diagonal(v[i], b.row(i) - b.col());
                        if (b.on_diagonal(i) && b.row(i) < g.rows) g.diag_out[diag + b.row(i)] = d * (1.f / (kUnitA * kUnitA)) + row_value[i] * g.diag_in2[diag + b.row(i)];
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[i][j] = row_value[i] * h[j] + f[j] * col_value[c & 1][j] + v[i][j] * (1.f / kUnitA);      // in kUnitA
                }
                store_symmetric(g, staging, t.g, b, v, t.mirror);
            } else {
                finish_update(g, staging, t.g, b, v, old[c & 1], low[c & 1], row_value);
            }
        }
        umma::fence_before_thread_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&s.sm->acc_empty[acc]);
        acc ^= 1;
        acc_phase ^= acc == 0;
    }
    return true;
}

template <int kBlockN>
__device__ __forceinline__ uint32_t ns_setup(const NsShared<kBlockN>& s) {
    if (threadIdx.x == 0) {
        for (int i = 0; i < NsShared<kBlockN>::kStages; ++i) {
            ptx::mbar_init(&s.sm->full[i], 1);
            ptx::mbar_init(&s.sm->empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&s.sm->acc_full[i], 1);
            ptx::mbar_init(&s.sm->acc_empty[i], kEpiWarps);
        }
        ptx::mbar_init(&s.sm->quiet, 1);
        s.sm->failed = 0;
        ptx::mbar_fence_init();
    }
    if (threadIdx.x >> 5 == 1) {
        umma::tmem_alloc(&s.sm->tmem_base, ns_tmem_columns(kBlockN));
        umma::tmem_relinquish();
    }
    umma::fence_before_thread_sync();
    __syncthreads();
    umma::fence_after_thread_sync();
    return s.sm->tmem_base;
}
// Where a wait has run out (which nobody can come to any more), what is still under way ends before its memory goes to others: what was requested has landed, and products
// have ended, those too that were issued before the wait ran out elsewhere.
template <class Landed>
__device__ __forceinline__ void ns_settle(NsSmem* sm, Landed landed) {
    __syncthreads();
    if (sm->failed == 0) return;
    const int warp = threadIdx.x >> 5;
    if (warp < 2 && ptx::elect_one()) {                // (the thread that requested, or issued)
        if (warp == 0) {
            landed();
        } else {
            umma::mma_commit(&sm->quiet);
            mbar_drain(&sm->quiet, 0, 1000000000ull);
        }
    }
    __syncthreads();
}

// One product of one step: a persistent CTA per SM, a warp that requests operands, one that issues the products, eight that finish tiles while the next one's products run
// (two accumulators).  Bound by the tensor cores and, in long runs, by power: 8 x 4096 x 7168 alone takes 707 us for X X^T, 413 for a product of squares (half of either
// is computed) and 1490 for X, 1.3 to 1.4 PFLOP/s; all 16 products of five steps, behind the norm and the cast, 15.1 ms, 1.06 PFLOP/s.  4 x 2048 x 3584: tensor pipe 72 % busy for X X^T and X, 53 to 59 % for squares
// (tiles of 32 K blocks).  Below some 1000 rows the chain of launches is what counts: 3 x 777 x 1001 takes 154 us in 17 launches, 34 GFLOP; all steps in one launch whose
// CTAs wait for one another took 237 (183 without), parts along K in a cluster's shared memory 145 for 256 x 7168 (121 without).
template <int kMode, int kBlockN>
__global__ void __launch_bounds__(kNsThreads, 1)
ns_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ NsArgs g) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const NsShared<kBlockN> s(smem);
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        umma::prefetch_tensormap(&map_a);
        umma::prefetch_tensormap(&map_b);
    }
    const uint32_t tmem_base = ns_setup(s);
    ptx::wait_for_previous_kernel();
    int acc = 0;
    uint32_t acc_phase = 0;
    NsRing<kBlockN> p;
    int loads = 0;
    if (warp == 0) {
        if (ptx::elect_one()) {
            ns_load<kMode, kBlockN>(g, s, &map_a, &map_b, p, loads);
            ptx::let_next_kernel_start();
        }
    } else if (warp == 1) {
        if (ptx::elect_one()) ns_multiply<kMode, kBlockN>(g, s, tmem_base, p, acc, acc_phase);
    } else {
        ns_finish<kMode, kBlockN>(g, s, tmem_base, acc, acc_phase);
    }
    umma::fence_before_thread_sync();
    ns_settle(s.sm, [&] { ns_drain(s, p, loads); });
    if (warp == 1) umma::tmem_dealloc(tmem_base, ns_tmem_columns(kBlockN));
}

// Short matrices: Q and X <- Q X in one kernel, a CTA per 128 x 128 tile of X, which makes the 128 rows of B that it needs itself and writes them over those of O, as the first
// operand of its second product.  One launch less per step, which is what these matrices take.
// Five steps with and without, in us: 64 x 64 47 and 60, 256 x 256 80 and 92, 256 x 7168 111 and 120, 32 of 256 x 256 93 and 111.
template <int kRows>
struct NsStepShared {
    static constexpr int kBlocks = kRows / kTileK, kBlockBytes = kRows * 128, kBytesX = kTileM * 128;       // blocks of 64 columns of O, of 64 rows of X
    uint8_t *o, *x, *staging;
    NsSmem* sm;
    float* coef;                                       // [128] the diagonal of Q
    __device__ __forceinline__ explicit NsStepShared(uint8_t* smem)
        : o(smem), x(smem + kBlocks * kBlockBytes), staging(x + kBlocks * kBytesX + 1024), sm(reinterpret_cast<NsSmem*>(x + kBlocks * kBytesX)),
          coef(reinterpret_cast<float*>(x + kBlocks * kBytesX + 512)) {}
    static constexpr int kBytes = kBlocks * (kBlockBytes + kBytesX) + 1024 + kEpiWarps * kStagingBytes;
    // eight neighbouring values of O or B
    __device__ __forceinline__ uint4* at(int row, int col) const {
        return reinterpret_cast<uint4*>(o + (col / kTileK) * kBlockBytes + row * 128 + ((((col % kTileK) / 8) ^ (row & 7)) * 16));
    }
};
template <int kRows>
__device__ __forceinline__ bool ns_step_multiply(const NsArgs& g, const NsStepShared<kRows>& s, uint32_t tmem_base, int m, int num_k) {
    constexpr uint32_t kSquare = umma::make_instr_desc(kTileM, kRows, umma::kFormatF16), kWide = umma::make_instr_desc(kTileM, kTileM, umma::kFormatF16, false, true);
    auto mine = [&](int kb) { return umma::make_smem_desc_sw128(s.o + kb * s.kBlockBytes + m * kTileM * 128); };
    if (!ns_wait(&s.sm->full[0], 0, s.sm, g.report, 4)) return false;
    umma::fence_after_thread_sync();
    for (int kb = 0; kb < num_k; ++kb) {
        const uint64_t desc_b = umma::make_smem_desc_sw128(s.o + kb * s.kBlockBytes);
#pragma unroll
        for (int k = 0; k < kTileK / 16; ++k)
            umma::mma_ss<false>(tmem_base, umma::advance_desc_k(mine(kb), k * 32), umma::advance_desc_k(desc_b, k * 32), kSquare, kb != 0 || k != 0);
    }
    umma::mma_commit(&s.sm->acc_full[0]);
    if (!ns_wait(&s.sm->acc_empty[0], 0, s.sm, g.report, 2) || !ns_wait(&s.sm->full[1], 0, s.sm, g.report, 4)) return false;
    umma::fence_after_thread_sync();
    for (int kb = 0; kb < num_k; ++kb) {
        const uint64_t desc_b = umma::make_smem_desc_mn_sw128(s.x + kb * s.kBytesX);
#pragma unroll
        for (int k = 0; k < kTileK / 16; ++k)
            umma::mma_ss<false>(tmem_base + kRows, umma::advance_desc_k(mine(kb), k * 32), umma::advance_desc_k(desc_b, k * 16 * 128), kWide, kb != 0 || k != 0);
    }
    umma::mma_commit(&s.sm->acc_full[1]);
    return true;
}
template <int kRows>
__device__ __forceinline__ void ns_step_finish(const NsArgs& g, const NsStepShared<kRows>& s, uint32_t tmem_base, const NsTile& t) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = warp & 3, half = (warp - 2) >> 2;
    uint8_t* staging = s.staging + (warp - 2) * kStagingBytes;
    const uint32_t tmem = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
    const float* diag = g.diag_in + static_cast<int64_t>(t.g) * g.ld_sq;
    const int64_t wide = static_cast<int64_t>(t.g) * g.rows * g.ld_x;
    const int row0 = t.m * kTileM + quad * 32;
    auto sums = [&](uint32_t column, float (&v)[4][8]) {
        uint32_t r[32];
        umma::tmem_ld_32x32(tmem + column, r);
        umma::tmem_ld_wait();
        spread(staging, r, v);
    };
    float di[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = row0 + i * 8 + (lane >> 2);
        di[i] = row < g.rows ? diag[row] : 0.f;
    }
    // (O itself as well: its values are read here)
    bool ok = __all_sync(0xffffffffu, ns_wait(&s.sm->full[0], 0, s.sm, g.report, 4) && ns_wait(&s.sm->acc_full[0], 0, s.sm, g.report, 5));
    umma::fence_after_thread_sync();
    if (ok) {
#pragma unroll 1
        for (int c = 0; c < kRows / 64; ++c) {
            const Block b{row0, half * (kRows / 2) + c * 32};
            float dj[8], v[4][8];
#pragma unroll
            for (int j = 0; j < 8; ++j) dj[j] = b.col() + j < g.rows ? diag[b.col() + j] : 0.f;
            sums(b.col0, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint4* at = s.at(b.row(i), b.col());
                float f[8];
                unpack_half(*at, f);
                const float coefficient = g.b + g.c * di[i];
                if (b.row0 == b.col0) {
                    const float d = take_diagonal(v[i], b.row(i) - b.col());
                    if (b.on_diagonal(i)) s.coef[quad * 32 + i * 8 + (lane >> 2)] = b.row(i) < g.rows ? g.a + g.b * di[i] + g.c * (di[i] * di[i] + d * (1.f / (kUnitA * kUnitA))) : 0.f;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = (coefficient + g.c * dj[j]) * f[j] + g.c * (1.f / kUnitA) * v[i][j];
                *at = make_uint4(pack_half(v[i][0], v[i][1]), pack_half(v[i][2], v[i][3]), pack_half(v[i][4], v[i][5]), pack_half(v[i][6], v[i][7]));
            }
        }
        ptx::fence_proxy_async_smem();
        umma::fence_before_thread_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&s.sm->acc_empty[0]);
    }
    // the old X, and the diagonal that other warps have made.  (Every warp comes here, whatever became of its wait.)
    uint4 old[2][4], low[2][4];
    auto block = [&](int c) { return Block{row0, t.n * kTileM + half * 64 + c * 32}; };
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const Block b = block(c);
            const bool in = b.row(i) < g.rows && b.col() < g.ld_x;
            const int64_t at = wide + static_cast<int64_t>(b.row(i)) * g.ld_x + b.col();
            old[c][i] = in ? *reinterpret_cast<const uint4*>(g.x_in + at) : make_uint4(0, 0, 0, 0);
            low[c][i] = in ? *reinterpret_cast<const uint4*>(g.x_lo + at) : make_uint4(0, 0, 0, 0);
        }
    asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarps * 32) : "memory");
    if (!ok) return;
    float q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = s.coef[quad * 32 + i * 8 + (lane >> 2)];
    ok = __all_sync(0xffffffffu, ns_wait(&s.sm->acc_full[1], 0, s.sm, g.report, 5));
    if (!ok) return;
    umma::fence_after_thread_sync();
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const Block b = block(c);
        if (b.row0 >= g.rows || b.col0 >= g.ld_x) break;
        float v[4][8];
        sums(kRows + half * 64 + c * 32, v);
        finish_update(g, staging, t.g, b, v, old[c], low[c], q);
    }
}
template <int kRows>
__global__ void __launch_bounds__(kNsThreads, 1)
ns_step_kernel(const __grid_constant__ CUtensorMap map_o, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ NsArgs g) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const NsStepShared<kRows> s(smem);
    constexpr int kColumns = kRows + kTileM <= 256 ? 256 : 512;
    const int warp = threadIdx.x >> 5, num_m = (g.rows + kTileM - 1) / kTileM, num_k = (g.rows + kTileK - 1) / kTileK;
    if (threadIdx.x == 0) {
        umma::prefetch_tensormap(&map_o);
        umma::prefetch_tensormap(&map_x);
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&s.sm->full[i], 1);
            ptx::mbar_init(&s.sm->acc_full[i], 1);
        }
        ptx::mbar_init(&s.sm->acc_empty[0], kEpiWarps);
        ptx::mbar_init(&s.sm->quiet, 1);
        s.sm->failed = 0;
        ptx::mbar_fence_init();
    }
    if (warp == 1) {
        umma::tmem_alloc(&s.sm->tmem_base, kColumns);
        umma::tmem_relinquish();
    }
    umma::fence_before_thread_sync();
    __syncthreads();
    umma::fence_after_thread_sync();
    const uint32_t tmem_base = s.sm->tmem_base;
    ptx::wait_for_previous_kernel();
    const NsTile t = ns_tile<kTileM, false>(blockIdx.x, num_m * ((g.cols + kTileM - 1) / kTileM), num_m);
    if (warp == 0) {
        if (ptx::elect_one()) {
            ptx::mbar_arrive_expect_tx(&s.sm->full[0], num_k * s.kBlockBytes);
            for (int kb = 0; kb < num_k; ++kb)
#pragma unroll
                for (int r = 0; r < kRows; r += kTileM) umma::tma_load_3d(s.o + kb * s.kBlockBytes + r * 128, &map_o, kb * kTileK, r, t.g, &s.sm->full[0]);
            ptx::mbar_arrive_expect_tx(&s.sm->full[1], num_k * s.kBytesX);
            for (int kb = 0; kb < num_k; ++kb)
#pragma unroll
                for (int i = 0; i < 2; ++i) umma::tma_load_3d(s.x + kb * s.kBytesX + i * umma::kMnChunkBytes, &map_x, t.n * kTileM + i * 64, kb * kTileK, t.g, &s.sm->full[1]);
            ptx::let_next_kernel_start();
        }
    } else if (warp == 1) {
        if (ptx::elect_one()) ns_step_multiply(g, s, tmem_base, t.m, num_k);
    } else {
        ns_step_finish(g, s, tmem_base, t);
    }
    umma::fence_before_thread_sync();
    ns_settle(s.sm, [&] {
        mbar_drain(&s.sm->full[0], 0, 1000000000ull);
        mbar_drain(&s.sm->full[1], 0, 1000000000ull);
    });
    if (warp == 1) umma::tmem_dealloc(tmem_base, kColumns);
}

// Eight rows of 32 values of a tile: the parts of X X^T added in their order, eight requested at a time.  Many small pieces, since what this takes is the way of the parts
// through L2.
template <int kBlockN>
struct NsAdd {
    static constexpr int kPieces = (kTileM / 8) * (kBlockN / 32);      // of a tile
};
template <int kBlockN>
__device__ __forceinline__ void ns_add_piece(const NsArgs& g, uint8_t* staging, int tile, int piece, int per_matrix, int num_tiles) {
    const int lane = threadIdx.x & 31;
    const NsTile t = ns_tile<kBlockN, true>(tile, per_matrix, 0);
    const int r = piece / (kBlockN / 32) * 8 + (lane >> 2), c = piece % (kBlockN / 32) * 32 + (lane & 3) * 8;
    const int row0 = t.m * kTileM + piece / (kBlockN / 32) * 8, col0 = t.n * kBlockN + piece % (kBlockN / 32) * 32, row = t.m * kTileM + r, col = t.n * kBlockN + c;
    if (row0 >= g.rows || col0 >= g.ld_sq) return;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    const float* part = g.parts + (static_cast<int64_t>(tile) * kTileM + r) * kBlockN + c;
    const int64_t pitch = static_cast<int64_t>(num_tiles) * kTileM * kBlockN;
    for (int s0 = 0; s0 < g.k_splits; s0 += 8) {
        float4 x[8], y[8];
#pragma unroll
        for (int s = 0; s < 8; ++s)
            if (s0 + s < g.k_splits) {
                x[s] = *reinterpret_cast<const float4*>(part + (s0 + s) * pitch);
                y[s] = *reinterpret_cast<const float4*>(part + (s0 + s) * pitch + 4);
            }
#pragma unroll
        for (int s = 0; s < 8; ++s)
            if (s0 + s < g.k_splits) {
                v[0] += x[s].x, v[1] += x[s].y, v[2] += x[s].z, v[3] += x[s].w;
                v[4] += y[s].x, v[5] += y[s].y, v[6] += y[s].z, v[7] += y[s].w;
            }
    }
    if (row0 >= col0 && row0 < col0 + 32) {
        const float d = take_diagonal(v, row - col);
        if (static_cast<uint32_t>(row - col) < 8u && row < g.rows) g.diag_out[static_cast<int64_t>(t.g) * g.ld_sq + row] = d * (1.f / (kUnitX * kUnitX));
    }
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = pack_half(v[2 * j] * (kUnitA / (kUnitX * kUnitX)), v[2 * j + 1] * (kUnitA / (kUnitX * kUnitX)));
    __half* out = g.sq_out + static_cast<int64_t>(t.g) * g.rows * g.ld_sq;
    if (row < g.rows && col < g.ld_sq) *reinterpret_cast<uint4*>(out + static_cast<int64_t>(row) * g.ld_sq + col) = make_uint4(o[0], o[1], o[2], o[3]);
    if (t.mirror) {
        // the mirror image: 32 rows of eight values
#pragma unroll
        for (int j = 0; j < 8; ++j) *reinterpret_cast<uint16_t*>(staging + ((lane & 3) * 8 + j) * 16 + (lane >> 2) * 2) = static_cast<uint16_t>(o[j >> 1] >> (16 * (j & 1)));
        __syncwarp();
        if (col0 + lane < g.rows && row0 < g.ld_sq)
            *reinterpret_cast<uint4*>(out + static_cast<int64_t>(col0 + lane) * g.ld_sq + row0) = *reinterpret_cast<const uint4*>(staging + lane * 16);
        __syncwarp();
    }
}

// Adds the parts of X X^T: a warp per piece of 8 rows x 32 columns, eight parts requested at once.  256 x 7168, 13 parts: 5 us
constexpr int kAddThreads = 128;
template <int kBlockN>
__global__ void __launch_bounds__(kAddThreads) ns_add_kernel(const __grid_constant__ NsArgs g) {
    __shared__ __align__(16) uint8_t s_staging[kAddThreads / 32][512];
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const int per_matrix = symmetric_tiles<kBlockN>(g.rows), num_tiles = per_matrix * g.count;
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kAddThreads / 32) + (threadIdx.x >> 5);
    constexpr int kPieces = NsAdd<kBlockN>::kPieces;
    if (unit < static_cast<int64_t>(num_tiles) * kPieces)
        ns_add_piece<kBlockN>(g, s_staging[threadIdx.x >> 5], static_cast<int>(unit / kPieces), static_cast<int>(unit % kPieces), per_matrix, num_tiles);
}

// ------------------------------------------------------------------------------------------------ the first X
constexpr int kNormThreads = 256, kCastTile = 64;

template <class T>
__device__ __forceinline__ float as_float(T v) {
    if constexpr (sizeof(T) == 2) return __bfloat162float(v);
    else return v;
}
// kWide: lines start on 16 bytes
template <class T, bool kWide>
__device__ __forceinline__ void load_values(const T* p, int n, float* v) {     // 16 / sizeof(T) values, the first n of them there
    constexpr int kPer = 16 / sizeof(T);
    if (kWide && n >= kPer) {
        T raw[kPer];
        *reinterpret_cast<uint4*>(raw) = *reinterpret_cast<const uint4*>(p);
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = as_float(raw[i]);
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = i < n ? as_float(p[i]) : 0.f;
    }
}

// sums of squares, in 64 bits (squares of small or large fp32 values leave the range of 32): one per CTA.  4 x 2048 x 3584 bf16: 23 us, 2.6 TB/s
template <class T, bool kWide>
__global__ void __launch_bounds__(kNormThreads) ns_norm_kernel(const __grid_constant__ NsArgs g) {
    __shared__ double s_sum[kNormThreads / 32];
    constexpr int kPer = 16 / sizeof(T);
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const T* src = reinterpret_cast<const T*>(g.in) + static_cast<int64_t>(blockIdx.y) * g.in_stride_matrix;
    double sum[2] = {0.0, 0.0};
    // pieces of a line, line after line
    const int per_line = (g.in_line + kPer - 1) / kPer;
    const int64_t pieces = g.in_lines * per_line, stride = static_cast<int64_t>(gridDim.x) * kNormThreads;
    int64_t at = static_cast<int64_t>(blockIdx.x) * kNormThreads + threadIdx.x, line = at / per_line;
    int piece = static_cast<int>(at - line * per_line);
    const int64_t line_step = stride / per_line;
    const int piece_step = static_cast<int>(stride - line_step * per_line);
#pragma unroll 4
    for (; at < pieces; at += stride) {
        float v[kPer];
        load_values<T, kWide>(src + line * g.in_stride_line + piece * kPer, g.in_line - piece * kPer, v);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const double d = v[i];
            sum[i & 1] = fma(d, d, sum[i & 1]);
        }
        line += line_step;
        piece += piece_step;
        if (piece >= per_line) piece -= per_line, ++line;
    }
    double total = sum[0] + sum[1];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = total;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kNormThreads / 32; ++w) total += s_sum[w];
        g.norm_parts[static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x] = total;
    }
}

// X = G / (norm + eps) as hi + lo, with rows <= cols; lines of the input are rows of X, or (flip) its columns.  One CTA per 64 x 64 tile,
// turned over in shared memory.  4 x 2048 x 3584 bf16: 37 us, 4.8 TB/s
template <class T, bool kWide>
__global__ void __launch_bounds__(kNormThreads) ns_cast_kernel(const __grid_constant__ NsArgs g) {
    __shared__ float tile[kCastTile][kCastTile + 1];
    __shared__ double s_scale;
    constexpr int kPer = 16 / sizeof(T), kPerLine = kCastTile / kPer;
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const int line0 = blockIdx.y * kCastTile, at0 = blockIdx.x * kCastTile;
    const T* src = reinterpret_cast<const T*>(g.in) + static_cast<int64_t>(blockIdx.z) * g.in_stride_matrix;
#pragma unroll
    for (int i = 0; i < kCastTile * kPerLine / kNormThreads; ++i) {
        const int u = i * kNormThreads + threadIdx.x, l = u / kPerLine, c = (u % kPerLine) * kPer;
        float v[kPer];
        load_values<T, kWide>(src + (line0 + l) * g.in_stride_line + at0 + c, line0 + l < g.in_lines ? g.in_line - at0 - c : 0, v);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (g.flip) tile[c + j][l] = v[j];
            else tile[l][c + j] = v[j];
        }
    }
    if (threadIdx.x < 32) {
        double sum = 0.0;
        for (int i = threadIdx.x; i < g.num_norm_parts; i += 32) sum += g.norm_parts[static_cast<int64_t>(blockIdx.z) * g.num_norm_parts + i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (threadIdx.x == 0) s_scale = static_cast<double>(kUnitX) / (sqrt(sum) + static_cast<double>(g.eps));
    }
    __syncthreads();
    const double scale = s_scale;
    // (a factor that is an ordinary 32-bit number serves as one)
    const float scale32 = static_cast<float>(scale);
    const bool ordinary = scale32 > 1e-30f && scale32 < 1e30f;
    const int row0 = g.flip ? at0 : line0, col0 = g.flip ? line0 : at0;
#pragma unroll
    for (int i = 0; i < kCastTile * kCastTile / 8 / kNormThreads; ++i) {
        const int u = i * kNormThreads + threadIdx.x, r = u / (kCastTile / 8), c = (u % (kCastTile / 8)) * 8;
        if (row0 + r < g.rows && col0 + c < g.ld_x) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float a = tile[r][c + 2 * j], b = tile[r][c + 2 * j + 1];
                const float x = ordinary ? a * scale32 : static_cast<float>(a * scale), y = ordinary ? b * scale32 : static_cast<float>(b * scale);
                hi[j] = pack_half(x, y);
                const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi[j]));
                lo[j] = pack_half((x - h.x) * kUnitLo, (y - h.y) * kUnitLo);
            }
            const int64_t at = (static_cast<int64_t>(blockIdx.z) * g.rows + row0 + r) * g.ld_x + col0 + c;
            *reinterpret_cast<uint4*>(g.x_out + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(g.x_lo + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
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

int64_t symmetric_tiles_of(int rows, int block_n) { return block_n == 256 ? symmetric_tiles<256>(rows) : symmetric_tiles<128>(rows); }
int64_t tiles_of(const NsArgs& g, int mode, int block_n) {
    return g.count * (mode == kUpdate ? static_cast<int64_t>((g.rows + kTileM - 1) / kTileM) * ((g.cols + block_n - 1) / block_n) : symmetric_tiles_of(g.rows, block_n));
}
// Columns of a tile: of 256, 128 and for X, whose tiles need not meet the diagonal, 192, the one whose waves take the least time, if a tile of 128 columns takes 0.6 and one of
// 192 takes 0.8 of one of 256; the wider one of equals.
int block_n_of(const NsArgs& g, int mode, int num_sms) {
    int best = 256;
    int64_t least = 0;
    for (int n = 256; n >= 128; n -= mode == kUpdate ? 64 : 128) {
        const int64_t time = (tiles_of(g, mode, n) + num_sms - 1) / num_sms * (n / 32 + 2);
        if (n == 256 || time < least) best = n, least = time;
    }
    return best;
}
// Parts along K of X X^T where its tiles are few and long: as in the GEMM, the K blocks that a CTA is spared against the kernel that adds the parts
// (about 16 blocks) and the parts' way through L2 (one block per 512 KB).
int k_splits_of(const NsArgs& g, int num_sms) {
    const int64_t tiles = tiles_of(g, kGram, 128), num_k = (g.cols + kTileK - 1) / kTileK, most = std::min<int64_t>(num_sms / tiles, num_k / 4);
    int64_t best = 1, gain = 0;
    for (int64_t s = 2; s <= most; ++s) {
        const int64_t now = num_k - (num_k + s - 1) / s - 16 - s * tiles * kTileM * 128 * 4 / (512 * 1024);
        if (now > gain) best = s, gain = now;
    }
    return static_cast<int>(best);
}

cudaError_t allow_smem(const void* fn, int bytes) {
    const cudaError_t err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err != cudaSuccess) cudaGetLastError();      // the caller reports it
    return err;
}
// ... once per device: a step has few launches, and they are what small matrices take
cudaError_t allow_once(const void* fn, int bytes, std::atomic<uint64_t>& allowed) {
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) return err;
    if (device >= 64 || (allowed.load(std::memory_order_relaxed) >> device & 1) == 0) {
        err = allow_smem(fn, bytes);
        if (err == cudaSuccess && device < 64) allowed.fetch_or(1ull << device, std::memory_order_relaxed);
    }
    return err;
}
template <int kMode, int kBlockN>
cudaError_t launch_product(const CUtensorMap& map_a, const CUtensorMap& map_b, const NsArgs& g, int num_sms, cudaStream_t stream) {
    const void* fn = reinterpret_cast<const void*>(ns_kernel<kMode, kBlockN>);
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t err = allow_once(fn, ns_smem_bytes(kBlockN), allowed);
    if (err != cudaSuccess) return err;
    const int64_t items = tiles_of(g, kMode, kBlockN) * (kMode == kGramPart ? g.k_splits : 1);
    void* params[] = {const_cast<CUtensorMap*>(&map_a), const_cast<CUtensorMap*>(&map_b), const_cast<NsArgs*>(&g)};
    return launch_dependent(fn, dim3(static_cast<unsigned>(std::min<int64_t>(items, num_sms))), dim3(kNsThreads), params, ns_smem_bytes(kBlockN), stream);
}
template <int kMode>
cudaError_t launch_product(int block_n, const CUtensorMap& map_a, const CUtensorMap& map_b, const NsArgs& g, int num_sms, cudaStream_t stream) {
    if constexpr (kMode == kUpdate)
        if (block_n == 192) return launch_product<kMode, 192>(map_a, map_b, g, num_sms, stream);
    return block_n == 256 ? launch_product<kMode, 256>(map_a, map_b, g, num_sms, stream) : launch_product<kMode, 128>(map_a, map_b, g, num_sms, stream);
}

// Short matrices whose tiles of X have an SM each: more tiles would make the polynomial again and again
bool in_one_kernel(const NsArgs& g, int num_sms) { return g.rows <= 256 && tiles_of(g, kUpdate, kTileM) <= num_sms; }
template <int kRows>
cudaError_t launch_step(const CUtensorMap& map_o, const CUtensorMap& map_x, const NsArgs& g, cudaStream_t stream) {
    const void* fn = reinterpret_cast<const void*>(ns_step_kernel<kRows>);
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t err = allow_once(fn, NsStepShared<kRows>::kBytes, allowed);
    if (err != cudaSuccess) return err;
    void* params[] = {const_cast<CUtensorMap*>(&map_o), const_cast<CUtensorMap*>(&map_x), const_cast<NsArgs*>(&g)};
    return launch_dependent(fn, dim3(static_cast<unsigned>(tiles_of(g, kUpdate, kTileM))), dim3(kNsThreads), params, NsStepShared<kRows>::kBytes, stream);
}

// rows of 128 bytes: a box of rows that start elsewhere takes three times as long on its way into shared memory
int64_t round64(int64_t n) { return (n + 63) / 64 * 64; }

template <class T>
cudaError_t launch_first(const NsArgs& g, cudaStream_t stream) {
    const bool wide = reinterpret_cast<uintptr_t>(g.in) % 16 == 0 && g.in_stride_line * sizeof(T) % 16 == 0 && g.in_stride_matrix * sizeof(T) % 16 == 0;
    void* params[] = {const_cast<NsArgs*>(&g)};
    const cudaError_t err = launch_dependent(wide ? reinterpret_cast<const void*>(ns_norm_kernel<T, true>) : reinterpret_cast<const void*>(ns_norm_kernel<T, false>),
                                             dim3(g.num_norm_parts, g.count), dim3(kNormThreads), params, 0, stream);
    if (err != cudaSuccess) return err;
    const dim3 grid((g.in_line + kCastTile - 1) / kCastTile, static_cast<unsigned>((g.in_lines + kCastTile - 1) / kCastTile), g.count);
    return launch_dependent(wide ? reinterpret_cast<const void*>(ns_cast_kernel<T, true>) : reinterpret_cast<const void*>(ns_cast_kernel<T, false>), grid, dim3(kNormThreads), params, 0,
                            stream);
}

// The largest singular value that X can have before any of `steps` steps: 1 before the first one (its squares add up to 1), then the largest
// |s (a + b s^2 + c s^4)| of s from 0 to it, a thousandth more for what rounding adds.  (The larger it is, the larger is the next one: they rise, or fall from the first on.)
double largest_singular_value(const NsArgs& g, int steps) {
    const double a = g.a, b = g.b, c = g.c;
    double top = 1.001;
    for (int i = 1; i < steps; ++i) {
        double next = 0.0;
        auto look = [&](double y) {                    // at s^2 = y
            if (y >= 0.0 && y <= top * top) next = std::max(next, std::sqrt(y) * std::abs(a + (b + c * y) * y));
        };
        look(top * top);
        // where the derivative 5 c y^2 + 3 b y + a is zero
        if (c == 0.0) {
            if (b != 0.0) look(-a / (3.0 * b));
        } else if (const double d = 9.0 * b * b - 20.0 * a * c; d >= 0.0) {
            look((-3.0 * b + std::sqrt(d)) / (10.0 * c));
            look((-3.0 * b - std::sqrt(d)) / (10.0 * c));
        }
        if (next >= 1e3) return 1e3;
        if (1.001 * next <= top) break;
        top = 1.001 * next;
    }
    return top;
}

// The first two steps as a pair: for matrices of half as many columns again as rows, if that saves more products than its additional kernel costs, and the matrices have rows
// enough for the rounding of a pair to stay below that of the result.  In us, five single steps and with a pair: 1024 x 1536 138 and 149, 1024 x 2048 147 and 157, four of them 238 and
// 236, eight 438 and 417, 16 of 512 x 2048 427 and 376, 1024 x 7168 250 and 238, 2048 x 7168 535 and 484, four of them 1910 and 1715; four of 2048 x 2560 (a quarter more) 855 and 850.
// Coefficients under which Q could grow past what fp16 holds of a product of two (64 beside the diagonal) stay with single steps.
bool first_pair(const NsArgs& g) {
    const double s = largest_singular_value(g, 2);
    const float top = static_cast<float>(std::max(1.5, s * s));              // eigenvalues of A, and of Q1 A Q1, are 0 to this
    auto small = [&](float x) { return std::abs(g.a + (g.b + g.c * x) * x) <= 4.f; };
    const float vertex = g.c == 0.f ? 0.f : std::min(std::max(-g.b / (2.f * g.c), 0.f), top);
    if (!small(0.f) || !small(top) || !small(vertex) || !(top <= 14.f)) return false;       // (T = Q1 A: 4 x 14)
    const int64_t saved = 3ll * (g.cols - g.rows) * g.rows * g.rows * g.count;       // multiply-adds
    return g.steps >= 2 && g.rows >= 512 && 2ll * g.cols >= 3ll * g.rows && saved >= 12'000'000'000;
}

}  // namespace

// What fp16 holds: 65504 / kUnitX of X's entries, which its largest singular value s bounds, and 65504 / kUnitA beside the diagonals of A and B, which half the range of their
// eigenvalues bounds: [0, s^2], and b y + c y^2 for y from 0 to s^2.
bool newton_schulz_fits(const NsArgs& g) {
    if (!std::isfinite(g.a) || !std::isfinite(g.b) || !std::isfinite(g.c)) return false;
    const double s = largest_singular_value(g, g.steps), y = s * s, limit = 60000.0;
    auto b_of = [&](double v) { return (g.b + static_cast<double>(g.c) * v) * v; };
    const double vertex = g.c == 0.f ? 0.0 : std::min(std::max(-g.b / (2.0 * g.c), 0.0), y);
    const double low = std::min({0.0, b_of(vertex), b_of(y)}), high = std::max({0.0, b_of(vertex), b_of(y)});
    return s * kUnitX <= limit && 0.5 * y * kUnitA <= limit && 0.5 * (high - low) * kUnitA <= limit;
}

// Workspace: hi of X twice and lo once, three symmetric matrices (two without a pair, one for short matrices) and their diagonals, sums of squares, parts of X X^T.
NsWorkspace newton_schulz_workspace(const NsArgs& g, int num_sms) {
    NsWorkspace w{};
    w.ld_x = round64(g.cols);
    w.ld_sq = round64(g.rows);
    w.norm_parts = std::max<int64_t>(1, std::min<int64_t>((static_cast<int64_t>(g.rows) * g.cols + 8191) / 8192, 8 * num_sms / g.count));
    w.k_splits = k_splits_of(g, num_sms);
    auto take = [&](int64_t bytes) {
        const int64_t at = w.bytes;
        w.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    w.norms = take(g.count * w.norm_parts * 8);
    for (int64_t& x : w.x) x = take(g.count * g.rows * w.ld_x * 2);
    w.lo = take(g.count * g.rows * w.ld_x * 2);
    for (int i = 0; i < (first_pair(g) ? 3 : in_one_kernel(g, num_sms) ? 1 : 2); ++i) {
        w.sq[i] = take(g.count * g.rows * w.ld_sq * 2);
        w.diag[i] = take(g.count * w.ld_sq * 4);
    }
    w.parts = take(w.k_splits > 1 ? w.k_splits * tiles_of(g, kGram, 128) * kTileM * 128 * 4 : 0);
    return w;
}

cudaError_t launch_newton_schulz(const NsArgs& args, const NsWorkspace& w, uint8_t* workspace, int num_sms, cudaStream_t stream) {
    const int steps = args.steps;
    if (args.count < 1 || args.rows < 1 || args.rows > args.cols || steps < 1 || !newton_schulz_fits(args) || reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return cudaErrorInvalidValue;
    NsArgs g = args;
    g.ld_x = static_cast<int>(w.ld_x);
    g.ld_sq = static_cast<int>(w.ld_sq);
    g.x_lo = reinterpret_cast<__half*>(workspace + w.lo);
    g.norm_parts = reinterpret_cast<double*>(workspace + w.norms);
    g.num_norm_parts = static_cast<int>(w.norm_parts);
    g.parts = reinterpret_cast<float*>(workspace + w.parts);
    g.k_splits = w.k_splits;
    g.out = nullptr;
    const bool pair_first = first_pair(g), one_kernel = in_one_kernel(g, num_sms);
    const int n_gram = g.k_splits > 1 ? 128 : block_n_of(g, kGram, num_sms), n_square = block_n_of(g, kPoly, num_sms), n_update = block_n_of(g, kUpdate, num_sms);
    // X in turn; symmetric matrices: their rows as the first and as the second operand
    struct Wide {
        __half* x;
        CUtensorMap rows, cols, mn;
    } x[2];
    struct Square {
        __half* m;
        float* diag;
        CUtensorMap rows, cols;
    } sq[3];
    for (int i = 0; i < 2; ++i) {
        x[i].x = reinterpret_cast<__half*>(workspace + w.x[i]);
        if (!make_map(&x[i].rows, x[i].x, g.count, g.rows, g.cols, g.ld_x, kTileM) || !make_map(&x[i].mn, x[i].x, g.count, g.rows, g.cols, g.ld_x, 64)) return cudaErrorInvalidValue;
        x[i].cols = x[i].rows;
        if (n_gram != kTileM && !make_map(&x[i].cols, x[i].x, g.count, g.rows, g.cols, g.ld_x, n_gram)) return cudaErrorInvalidValue;
    }
    for (int i = 0; i < (pair_first ? 3 : one_kernel ? 1 : 2); ++i) {
        sq[i].m = reinterpret_cast<__half*>(workspace + w.sq[i]);
        sq[i].diag = reinterpret_cast<float*>(workspace + w.diag[i]);
        if (!make_map(&sq[i].rows, sq[i].m, g.count, g.rows, g.rows, g.ld_sq, kTileM)) return cudaErrorInvalidValue;
        sq[i].cols = sq[i].rows;
        if (n_square != kTileM && !make_map(&sq[i].cols, sq[i].m, g.count, g.rows, g.rows, g.ld_sq, n_square)) return cudaErrorInvalidValue;
    }
    auto gram = [&](const Wide& from, const Square& to) {
        g.sq_out = to.m;
        g.diag_out = to.diag;
        if (g.k_splits == 1) return launch_product<kGram>(n_gram, from.rows, from.cols, g, num_sms, stream);
        const cudaError_t err = launch_product<kGramPart, 128>(from.rows, from.cols, g, num_sms, stream);
        if (err != cudaSuccess) return err;
        void* params[] = {&g};
        const int64_t warps = tiles_of(g, kGram, 128) * NsAdd<128>::kPieces;
        return launch_dependent(reinterpret_cast<const void*>(ns_add_kernel<128>), dim3(static_cast<unsigned>(warps * 32 / kAddThreads)), dim3(kAddThreads), params, 0, stream);
    };
    auto poly = [&](const Square& from, const Square& to) {
        g.sq_in = from.m;
        g.diag_in = from.diag;
        g.sq_out = to.m;
        g.diag_out = to.diag;
        return launch_product<kPoly>(n_square, from.rows, from.cols, g, num_sms, stream);
    };
    auto product = [&](const Square& p, const Square& r, const Square& to) {
        g.sq_in = p.m;
        g.diag_in = p.diag;
        g.sq_in2 = r.m;
        g.diag_in2 = r.diag;
        g.sq_out = to.m;
        g.diag_out = to.diag;
        return launch_product<kProduct>(n_square, p.rows, r.cols, g, num_sms, stream);
    };
    // X <- Q X, with Q of A
    auto step = [&](const Square& from_a, const Wide& from, const Wide& to) {
        g.diag_in = from_a.diag;
        g.x_in = from.x;
        g.x_out = to.x;
        return g.rows <= 128 ? launch_step<128>(from_a.rows, from.mn, g, stream) : launch_step<256>(from_a.rows, from.mn, g, stream);
    };
    auto update = [&](const Square& q, const Wide& from, const Wide& to) {
        g.diag_in = q.diag;
        g.x_in = from.x;
        g.x_out = to.x;
        return launch_product<kUpdate>(n_update, q.rows, from.mn, g, num_sms, stream);
    };

    g.x_out = x[0].x;
    cudaError_t err = g.in_bf16 ? launch_first<__nv_bfloat16>(g, stream) : launch_first<float>(g, stream);
    for (int done = 0, from = 0; done < steps && err == cudaSuccess; from ^= 1) {
        const bool pair = pair_first && done == 0;
        done += pair ? 2 : 1;
        err = gram(x[from], sq[0]);
        if (err == cudaSuccess && !one_kernel) err = poly(sq[0], sq[1]);
        if (pair) {
            if (err == cudaSuccess) err = product(sq[1], sq[0], sq[2]);      // T = Q1 A
            if (err == cudaSuccess) err = product(sq[2], sq[1], sq[0]);      // A = T Q1
            if (err == cudaSuccess) err = poly(sq[0], sq[2]);                // Q2
            if (err == cudaSuccess) err = product(sq[2], sq[1], sq[0]);      // Q = Q2 Q1
        }
        if (done == steps) g.out = args.out;
        if (err == cudaSuccess) err = one_kernel ? step(sq[0], x[from], x[from ^ 1]) : update(sq[pair ? 0 : 1], x[from], x[from ^ 1]);
    }
    return err;
}

}  // namespace ep
