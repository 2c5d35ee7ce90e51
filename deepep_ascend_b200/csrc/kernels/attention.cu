// Attention of packed sequences on the tensor cores, forward and backward.  Per sequence and query head, with the keys and values of its group,
//
//     S = scale Q K^T (only what a query sees),   P = softmax(S),   O = P V,   lse = log sum exp(S)
//     delta = rowsum(dO O) - d_lse,   dP = dO V^T,   dS = P (dP - delta)
//     dV = P^T dO,   dQ = scale dS K,   dK = scale dS^T Q        (dK, dV: over the heads of the group)
//
// Products are tcgen05 (bf16 operands, 32-bit sums in tensor memory).  The softmax is taken in one pass over the keys with a running reference and sum, all
// in 32 bits; P and dS are rounded to bf16, as operands of the products that follow (an unbiased 2^-9 of each term, which in a sum of many is less than
// the rounding of the result).
//
// A causal query sees the keys up to its own place, both sequences ending together: query i of nq the keys 0 .. nk - nq + i of nk.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "gemm_sm100.cuh"

namespace ep {

namespace {

constexpr uint64_t kAttnWaitLimitNs = 4ull * 1000 * 1000 * 1000;      // when the caller gives no limit
constexpr uint64_t kLandNs = 10ull * 1000 * 1000;                     // after a failure: what a copy is given to land (a phase that nothing is on its way for takes it all)
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

using bf16 = __nv_bfloat16;

// ------------------------------------------------------------------------------------------------ waits
struct AttnState {
    uint32_t tmem_base;
    int failed;
};
// Bounded wait for an mbarrier phase; when it runs out the device's flag is raised, and the status block of the caller's buffer written.
__device__ __noinline__ void attn_fail(const NsReport& r, int* failed, int code) {
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
// code: 1 free stage, 2 probabilities, 3 scores that have been read, 4 full stage, 5 scores, 6 sums and statistics, 7 work
__device__ __forceinline__ bool attn_wait(uint64_t* bar, uint32_t parity, int* failed, const NsReport& r, int code) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns(), limit = r.timeout_ns != 0 ? r.timeout_ns : kAttnWaitLimitNs;
    uint32_t spins = 0;
    while (!ptx::mbar_try_wait(bar, parity)) {
        if ((++spins & 63u) == 0u) {
            if (*reinterpret_cast<volatile int*>(failed)) return false;
            if (globaltimer_ns() - t0 > limit) {
                attn_fail(r, failed, code);
                return false;
            }
        }
    }
    return true;
}
// ... of a whole warp
__device__ __forceinline__ bool attn_wait_warp(uint64_t* bar, uint32_t parity, int* failed, const NsReport& r, int code) {
    return __all_sync(0xffffffffu, attn_wait(bar, parity, failed, r, code)) != 0;
}

template <int kStages>
struct AttnRing {
    int stage = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void advance() {
        if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
        }
    }
};

// ------------------------------------------------------------------------------------------------ work
// Blocks of `rows` rows of the sequences are numbered without a count of them: sequence i has the numbers from cu[i] / rows + i on, up to one more than it needs.
struct AttnBlock {
    int seq, row0, rows;             // first row of the block inside its sequence, rows of the sequence (row0 >= rows: no block has this number)
    int start;                       // first row of the sequence
};
__device__ __forceinline__ int2 sequence_rows(const int32_t* cu, int i, int total) {
    if (cu == nullptr) return make_int2(0, total);
    const int a = min(max(cu[i], 0), total), b = min(max(cu[i + 1], a), total);
    return make_int2(a, b - a);
}
__device__ __forceinline__ AttnBlock find_block(const int32_t* cu, int num_seqs, int total, int number, int rows) {
    int lo = 0;
    if (cu != nullptr) {
        int hi = num_seqs;                                        // the last i in [lo, hi) with cu[i] / rows + i <= number
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (min(max(cu[mid], 0), total) / rows + mid <= number) lo = mid;
            else hi = mid;
        }
    }
    const int2 s = sequence_rows(cu, lo, total);
    const int at = number - s.x / rows - lo;                     // (below zero: in front of the first sequence)
    return AttnBlock{lo, at < 0 ? s.y : at * rows, s.y, s.x};
}
int64_t num_blocks(int64_t total, int64_t num_seqs, int rows) { return total / rows + num_seqs; }

// kThreads threads: rows that belong to no sequence get zeros (and -inf), one of `parts` of them
template <int kThreads>
__device__ __forceinline__ void clear_rows(const int32_t* cu, int num_seqs, int total, int part, int parts, bf16* out, int64_t row_values, float* lse, int heads) {
    if (cu == nullptr) return;
    const int first = min(max(cu[0], 0), total), last = min(max(cu[num_seqs], first), total);
    const int missing = first + total - last;
    for (int i = part; i < missing; i += parts) {
        const int row = i < first ? i : last + i - first;
        for (int64_t c = threadIdx.x % kThreads; c < row_values / 8; c += kThreads) reinterpret_cast<uint4*>(out + row * row_values)[c] = make_uint4(0, 0, 0, 0);
        if (lse != nullptr)
            for (int h = threadIdx.x % kThreads; h < heads; h += kThreads) lse[static_cast<int64_t>(h) * total + row] = __int_as_float(0xff800000);
    }
}

// ------------------------------------------------------------------------------------------------ operands
// A tile of rows x 64 kChunks channels lies in shared memory as chunks of 64 channels, rows of 128 bytes with the 128-byte swizzle, as TMA writes them.  It is
// an operand along its channels (K-major) and along its rows (MN-major: every channel a row of the operand) alike.
// Lower halves of the descriptors (the upper ones, of eight rows per 1024 bytes, are all alike)
__device__ __forceinline__ uint32_t desc_channels(const uint8_t* tile) { return (ptx::smem_u32(tile) & 0x3ffffu) >> 4 | 1u << 16; }
template <int kRows>
__device__ __forceinline__ uint32_t desc_rows(const uint8_t* tile) { return (ptx::smem_u32(tile) & 0x3ffffu) >> 4 | static_cast<uint32_t>(kRows * 128 >> 4) << 16; }
__device__ __forceinline__ uint64_t desc_of(uint32_t low) { return static_cast<uint64_t>((1024u >> 4) | 1u << 14 | 2u << 29) << 32 | low; }
// D (+)= A B over the channels / over kSteps * 16 rows.  Descriptors step by constants and loops are unrolled: the one thread that issues products has 64 clocks for each.
template <int kRowsA, int kRowsB, int kChunks>
__device__ __forceinline__ void multiply_channels(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, int dim16) {
#pragma unroll
    for (int k = 0; k < 4 * kChunks; ++k)
        if (k < dim16)
            umma::mma_ss<false>(d, desc_of(a + ((k >> 2) * kRowsA * 128 + (k & 3) * 32) / 16), desc_of(b + ((k >> 2) * kRowsB * 128 + (k & 3) * 32) / 16), idesc, k != 0);
}
template <int kFirst, int kSteps>
__device__ __forceinline__ void multiply_rows(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
#pragma unroll
    for (int k = kFirst; k < kFirst + kSteps; ++k) umma::mma_ts(d, a + k * 8, desc_of(b + k * 16 * 128 / 16), idesc, add || k != 0);
}
template <int kRows, int kChunks>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, int head, int row, uint64_t* bar) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) umma::tma_load_3d(dst + c * kRows * 128, map, c * 64, head, row, bar);
}
// A warp: zeros in the rows from `valid` on, which belong to others and may hold anything: a probability of zero times an infinity is a NaN
template <int kRows, int kChunks>
__device__ __forceinline__ void clear_tile(uint8_t* tile, int valid) {
    const int lane = threadIdx.x & 31, pieces = (kRows - valid) * 8;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
        for (int i = lane; i < pieces; i += 32) *reinterpret_cast<uint4*>(tile + c * kRows * 128 + valid * 128 + i * 16) = make_uint4(0, 0, 0, 0);
    ptx::fence_proxy_async_smem();
    __syncwarp();
}

// ------------------------------------------------------------------------------------------------ numbers
__device__ __forceinline__ float exp2_approx(float x) {              // 2 ulp; 0 for -inf
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t v;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
    return v;
}
__device__ __forceinline__ uint64_t f32x2(float lo, float hi) { return umma::pack_f32x2(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
constexpr float kNone = -__builtin_huge_valf();
// (a NaN if one of them is)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// 2^x of a pair without the special function unit, which makes 16 a clock of an SM and would be what the softmax waits for: x = n + f with n the nearest whole number, 2^f
// by a polynomial of degree 4 (relative error 2.87e-6, least largest error on [-1/2, 1/2] with a constant of exactly 1, so that -127 and below give exactly 0), n added
// to the exponent.  A NaN may become any number: a row that has one is told by its largest score.
__device__ __forceinline__ uint64_t exp2_by_polynomial(uint64_t x2) {
    float x, y;
    umma::unpack_f32x2(x2, x, y);
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x));
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(y));
    x2 = f32x2(x, y);
    const uint64_t shift = f32x2(12582912.f, 12582912.f), back = f32x2(-12582912.f, -12582912.f), minus_one = f32x2(-1.f, -1.f);
    const uint64_t n = add2(x2, shift), f = fma2(add2(n, back), minus_one, x2);
    uint64_t p = fma2(f, f32x2(0.009585382388763709f, 0.009585382388763709f), f32x2(0.05590662825543393f, 0.05590662825543393f));
    p = fma2(p, f, f32x2(0.24024038166610448f, 0.24024038166610448f));
    p = fma2(p, f, f32x2(0.6931241843387045f, 0.6931241843387045f));
    p = fma2(p, f, f32x2(1.f, 1.f));
    float u, v, a, b;
    umma::unpack_f32x2(p, u, v);
    umma::unpack_f32x2(n, a, b);
    return umma::pack_f32x2(__float_as_uint(u) + (__float_as_uint(a) << 23), __float_as_uint(v) + (__float_as_uint(b) << 23));
}
constexpr int kPolynomialOf = 4;                     // of so many pairs of a row one goes by the polynomial

// The groups of four warps that hold rows take registers of the other one: 384 x 168 at launch = 128 x (2 rows' + the others'), 256 x 128 = 128 x (rows' + the others')
constexpr int kFwdRegisters = 224, kFwdRegistersOfTwo = 200, kBwdRegisters = 208;
template <int kRegisters>
__device__ __forceinline__ void take_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegisters));
}
template <int kRegisters>
__device__ __forceinline__ void give_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegisters));
}

// The first n of 32 bits
__device__ __forceinline__ uint32_t first_bits(int n) { return n >= 32 ? ~0u : (n <= 0 ? 0u : (1u << n) - 1u); }
// -inf where a bit is not set: bits become predicates several at a time (31 prompts of 264: 128 -> 125.5 us; in the backward pass, whose warps have half as many columns, it gave nothing)
__device__ __forceinline__ void hide(uint32_t (&s)[32], uint32_t bits) {
#pragma unroll
    for (int k = 0; k < 32; ++k) s[k] = bits >> k & 1u ? s[k] : 0xff800000u;
}
// A row of sums in tensor memory, times `factor`, as bf16
template <int kColumns>
__device__ __forceinline__ void store_row(uint32_t tmem, float factor, bf16* row, int dim, bool write) {
#pragma unroll
    for (int c = 0; c < kColumns; c += 32) {
        uint32_t r[32];
        umma::tmem_ld_32x32(tmem + c, r);
        umma::tmem_ld_wait();
        uint32_t v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = pack_bf16(__uint_as_float(r[2 * i]) * factor, __uint_as_float(r[2 * i + 1]) * factor);
        // (32 bytes at once, a sector, where rows start on them)
        if (dim % 16 == 0) {
#pragma unroll
            for (int i = 0; i < 16; i += 8)
                if (write && c + 2 * i < dim)
                    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(row + c + 2 * i), "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]),
                                 "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
                                 : "memory");
        } else {
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                if (write && c + 2 * i < dim) *reinterpret_cast<uint4*>(row + c + 2 * i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
    }
}

// ... as it is, in 32 bits
template <int kColumns>
__device__ __forceinline__ void store_part(uint32_t tmem, float factor, float* row, int dim, bool write) {
#pragma unroll
    for (int c = 0; c < kColumns; c += 32) {
        uint32_t r[32];
        umma::tmem_ld_32x32(tmem + c, r);
        umma::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; i += 4)
            if (write && c + i < dim)
                *reinterpret_cast<float4*>(row + c + i) = make_float4(__uint_as_float(r[i]) * factor, __uint_as_float(r[i + 1]) * factor, __uint_as_float(r[i + 2]) * factor,
                                                                      __uint_as_float(r[i + 3]) * factor);
    }
}

// ------------------------------------------------------------------------------------------------ forward
// A CTA takes two tiles of 128 queries that share keys and values, of two heads of a group or, where it has no second one, of one head, whose softmaxes (four warps each, a row per thread) and products alternate: while one tile's scores are made into
// probabilities, the tensor cores work for the other.  Probabilities take the place of the scores in tensor memory, from where they are the first operand of the next product.
//
// A CTA goes on with the work of CTAs that have not started (it cancels their launch and takes their place): barriers and tensor memory are set up once, and the next block's
// queries, keys and values come while the last one's results leave.  Blocks differ in length, so who takes which is decided as they end.  (31 prompts of 264 tokens, 56 heads of 128: 268 us with
// a CTA for every block, 150 so at the time.)
//
// Long sequences are bound by power: 16384 tokens, 56 heads of 128, 3.0 to 3.5 ms, 1.1 to 1.3 PFLOP/s at SM clocks of 1.4 to 1.55 GHz, the tensor pipe busy in 67 % of them.  What the clocks go by is the
// chain of a tile's block of 128 keys, some 3000 of which two tiles share: 70 for the scores into registers, 370 for their largest, 1050 for the powers, 100 for their way back, 512 + 512 for
// the products and as much for the barriers between, which lie in the shared memory that the products read at its full rate.  So a quarter of the powers by polynomial, the first half of
// the probabilities handed over early and an issuing thread for each tile took it from 3650 clocks to 3030.
// Small tasks have one tile per CTA and two CTAs on an SM, one of which works while the other begins or ends a block; two tiles read keys and values from L2 once for both.
// That tile takes the heads of a group together, each of as many queries as fill 128 rows (7 heads: 18), so that few rows stay empty where a sequence ends: 31 prompts of 264 tokens
// 125 -> 90 us (to 103 on other GPUs), 200 of 30 tokens (32 heads) 97 -> 46, 8 of 1000 152 either way.
constexpr int kPackedHeads = 16;
template <int kChunks, int kTiles>
struct FwdShape {
    // four warps per tile for its softmax; one that requests tiles, one per tile that issues products, one that looks for work, and to make up four more one without any
    static constexpr int kRowWarps = 4 * kTiles, kLoadWarp = kRowWarps, kMultiplyWarp = kRowWarps + 1, kWorkWarp = kRowWarps + 1 + kTiles;
    static constexpr int kThreads = kRowWarps * 32 + 128, kReaders = kRowWarps + 1 + kTiles, kRegisters = kTiles == 2 ? kFwdRegisters : kFwdRegistersOfTwo;
    static constexpr int kLaunchRegisters = kTiles == 2 ? 168 : 128;
    static constexpr int kTileBytes = 128 * 128 * kChunks, kStages = kTiles == 2 ? (kChunks == 2 ? 5 : 8) : (kChunks == 2 ? 2 : 5);
    static constexpr int kOut = kTiles * 128, kColumns = kTiles * 256;      // tensor memory: the tiles' scores, then their sums
    static constexpr int kSmem = (kTiles + kStages) * kTileBytes + 1024;
};
struct FwdWork {
    int start, rows;                 // as of AttnBlock; rows < 0: no more work
    int key0, keys, kv_head;
    int row0[2], head[2];            // of the tiles
    int n[2];                        // blocks of 128 keys that their rows see (0: there is nothing to do but to write zeros, if there are rows)
    __device__ __forceinline__ int blocks() const { return max(n[0], n[1]); }
};
struct FwdBars {
    alignas(16) uint4 answer;        // to the request for more work
    FwdWork work;
    uint64_t q_full[2], q_empty[2], full[8], empty[8], s_full[2], p_full[2][2], o_full[2], work_full, work_read, answered, tail, quiet[2];
    AttnState st;
};
// The next block of the grid that no CTA has started yet, or -1
template <class Bars>
__device__ __forceinline__ void request_work(Bars* b) {
    ptx::mbar_arrive_expect_tx(&b->answered, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(ptx::smem_u32(&b->answer)), "r"(ptx::smem_u32(&b->answered))
                 : "memory");
}
template <class Bars>
__device__ __forceinline__ int work_of_answer(Bars* b) {
    uint32_t x, got;
    asm volatile(
        "{\n .reg .pred p;\n .reg .b128 a;\n .reg .b32 y, z, w;\n ld.shared.b128 a, [%2];\n clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n"
        " selp.u32 %1, 1, 0, p;\n mov.u32 %0, 0;\n @p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, y, z, w}, a;\n}\n"
        : "=r"(x), "=r"(got)
        : "r"(ptx::smem_u32(&b->answer))
        : "memory");
    ptx::fence_proxy_async_smem();                   // (read before the next answer comes)
    return got != 0 ? static_cast<int>(x) : -1;
}

template <int kChunks, int kTiles>
__global__ void __launch_bounds__(FwdShape<kChunks, kTiles>::kThreads, 3 - kTiles)
attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                 const __grid_constant__ AttentionArgs a) {
    using Shape = FwdShape<kChunks, kTiles>;
    constexpr int kStages = Shape::kStages, kTileBytes = Shape::kTileBytes;
    const int pack = a.pack, tokens = 128 / pack;      // heads and tokens of a tile
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *sq = smem, *skv = smem + kTiles * kTileBytes;
    FwdBars* b = reinterpret_cast<FwdBars*>(smem + (kTiles + kStages) * kTileBytes);
    const int warp = threadIdx.x >> 5;
    int* failed = &b->st.failed;
    if (threadIdx.x == 0) {
        umma::prefetch_tensormap(&map_q);
        umma::prefetch_tensormap(&map_k);
        umma::prefetch_tensormap(&map_v);
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&b->q_full[i], 1);
            ptx::mbar_init(&b->q_empty[i], 1);
            ptx::mbar_init(&b->s_full[i], 1);
            ptx::mbar_init(&b->p_full[i][0], 4);
            ptx::mbar_init(&b->p_full[i][1], 4);
            ptx::mbar_init(&b->o_full[i], 1);
            ptx::mbar_init(&b->quiet[i], 1);
        }
        for (int i = 0; i < kStages; ++i) {
            ptx::mbar_init(&b->full[i], 1);
            ptx::mbar_init(&b->empty[i], kTiles);
        }
        ptx::mbar_init(&b->work_full, 1);
        ptx::mbar_init(&b->work_read, Shape::kReaders);
        ptx::mbar_init(&b->answered, 1);
        ptx::mbar_init(&b->tail, 1);
        b->st.failed = 0;
        ptx::mbar_fence_init();
    }
    if (warp == Shape::kMultiplyWarp) {
        umma::tmem_alloc(&b->st.tmem_base, Shape::kColumns);
        umma::tmem_relinquish();
    }
    if (warp == Shape::kLoadWarp)
        for (int t = 0; t < kTiles; ++t) clear_tile<128, kChunks>(sq + t * kTileBytes, tokens * pack);      // (rows that no query has)
    umma::fence_before_thread_sync();
    __syncthreads();
    umma::fence_after_thread_sync();
    const uint32_t tmem = b->st.tmem_base;
    ptx::wait_for_previous_kernel();
    // The k-th block of this CTA, for a whole warp; false: no more
    auto next_work = [&](int k, FwdWork& w) {
        if (!attn_wait_warp(&b->work_full, k & 1, failed, a.report, 7)) return false;
        w = b->work;
        __syncwarp();
        if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(&b->work_read);
        return w.rows >= 0;
    };

    if (warp >= Shape::kRowWarps) {
        give_registers<(kTiles + 1) * Shape::kLaunchRegisters - kTiles * Shape::kRegisters>();
        if (warp == Shape::kLoadWarp) {
            AttnRing<kStages> p;
            const bool one = ptx::elect_one();
            uint32_t tails = 0, queries[2] = {0, 0};
            FwdWork w;
            auto request = [&](const CUtensorMap* map, int j, bool clear) {
                if (!attn_wait_warp(&b->empty[p.stage], p.phase ^ 1, failed, a.report, 1)) return false;
                uint8_t* tile = skv + p.stage * kTileBytes;
                const bool tail = clear && j * 128 + 128 > w.keys;
                uint64_t* bar = tail ? &b->tail : &b->full[p.stage];
                if (one) {
                    ptx::mbar_arrive_expect_tx(bar, kTileBytes);
                    load_tile<128, kChunks>(tile, map, w.kv_head, w.key0 + j * 128, bar);
                }
                __syncwarp();
                if (tail) {
                    if (!attn_wait_warp(&b->tail, tails & 1, failed, a.report, 4)) return false;
                    ++tails;
                    clear_tile<128, kChunks>(tile, w.keys - j * 128);
                    if (one) ptx::mbar_arrive(&b->full[p.stage]);
                }
                p.advance();
                return true;
            };
            auto load = [&]() {
                for (int k = 0; next_work(k, w); ++k) {
                    const int blocks = w.blocks();
#pragma unroll
                    for (int t = 0; t < kTiles; ++t)
                        if (w.n[t] > 0) {
                            if (!attn_wait_warp(&b->q_empty[t], (queries[t] & 1) ^ 1, failed, a.report, 1)) return;
                            ++queries[t];
                            if (one) {
                                ptx::mbar_arrive_expect_tx(&b->q_full[t], tokens * pack * 128 * kChunks);
                                load_tile<128, kChunks>(sq + t * kTileBytes, &map_q, w.head[t], w.start + w.row0[t], &b->q_full[t]);
                            }
                            __syncwarp();
                        }
                    for (int j = 0; j < blocks; ++j)
                        if (!request(&map_k, j, false) || !request(&map_v, j, true)) return;
                }
            };
            load();
        } else if (warp < Shape::kWorkWarp) {
            // a tile's products; what no tile reads any more is free
            const int t = warp - Shape::kMultiplyWarp;
            const bool one = ptx::elect_one();
            const int dim16 = (a.dim + 15) / 16;
            const uint32_t idesc_s = umma::make_instr_desc(128, 128, umma::kFormatBF16), to_s = tmem + t * 128, to_o = tmem + Shape::kOut + t * 128;
            const uint32_t idesc_o = umma::make_instr_desc(128, 16, umma::kFormatBF16, false, true) + (static_cast<uint32_t>(2 * dim16 - 2) << 17);
            const uint32_t queries = desc_channels(sq + t * kTileBytes), keys_of = desc_channels(skv), values_of = desc_rows<128>(skv);
            auto free_stage = [&](int stage, bool read) {
                if (read) umma::mma_commit(&b->empty[stage]);
                else ptx::mbar_arrive(&b->empty[stage]);
            };
            AttnRing<kStages> p;
            uint32_t loads = 0, handed = 0;           // tiles of queries, blocks of probabilities so far
            auto scores = [&](bool last) {
                umma::fence_after_thread_sync();
                multiply_channels<128, 128, kChunks>(to_s, queries, keys_of + p.stage * (kTileBytes / 16), idesc_s, dim16);
                umma::mma_commit(&b->s_full[t]);
                if (last) umma::mma_commit(&b->q_empty[t]);
            };
            auto multiply = [&](int blocks, int mine) {
                if (!attn_wait(&b->full[p.stage], p.phase, failed, a.report, 4)) return;
                if (mine > 0) {
                    if (!attn_wait(&b->q_full[t], loads & 1, failed, a.report, 4)) return;
                    ++loads;
                    scores(mine == 1);
                }
                free_stage(p.stage, mine > 0);
                p.advance();
                for (int j = 0; j < blocks; ++j) {
                    // (the values, and the next keys, have mostly long been there)
                    const int stage_v = p.stage;
                    const uint32_t values = values_of + stage_v * (kTileBytes / 16);
                    if (!attn_wait(&b->full[stage_v], p.phase, failed, a.report, 4)) return;
                    p.advance();
                    if (j + 1 < blocks && !attn_wait(&b->full[p.stage], p.phase, failed, a.report, 4)) return;
                    if (j < mine) {
                        // the first half of the probabilities as soon as it is there
                        if (!attn_wait(&b->p_full[t][0], handed & 1, failed, a.report, 2)) return;
                        umma::fence_after_thread_sync();
                        multiply_rows<0, 4>(to_o, to_s, values, idesc_o, j != 0);
                        if (!attn_wait(&b->p_full[t][1], handed & 1, failed, a.report, 2)) return;
                        ++handed;
                        umma::fence_after_thread_sync();
                        multiply_rows<4, 4>(to_o, to_s, values, idesc_o, true);
                        if (j + 1 < mine) scores(j + 2 == mine);
                        else umma::mma_commit(&b->o_full[t]);
                    }
                    free_stage(stage_v, j < mine);
                    if (j + 1 < blocks) {
                        free_stage(p.stage, j + 1 < mine);
                        p.advance();
                    }
                }
            };
            FwdWork w;
            for (int k = 0; next_work(k, w); ++k) {
                if (one && w.blocks() > 0) multiply(w.blocks(), t == 0 ? w.n[0] : w.n[1]);
                __syncwarp();
            }
        } else if (warp == Shape::kWorkWarp) {
            // looks for work: first this CTA's own
            const int units = a.heads / pack, blocks = gridDim.x / units;
            int item = blockIdx.x;
            uint32_t handed = 0;
            bool something = true;
            for (uint32_t answers = 0;; ++answers) {
                FwdWork w{};
                w.rows = -1;
                if (item >= 0) {
                    // two tiles: 256 rows of a group's heads are as many pairs of tiles as the group has heads.  Long blocks first: those at the ends of the sequences
                    const int number = item / units, unit = item - number * units, group = a.heads / a.kv_heads / pack;
                    const AttnBlock blk = find_block(a.cu_q, a.num_seqs, a.tq, blocks - 1 - number, kTiles * tokens);
                    const int2 keys = sequence_rows(a.cu_k, blk.seq, a.tk);
                    clear_rows<32>(a.cu_q, a.num_seqs, a.tq, item, gridDim.x, reinterpret_cast<bf16*>(a.o), static_cast<int64_t>(a.heads) * a.dim, a.lse, a.heads);
                    w.start = blk.start;
                    w.rows = blk.rows;
                    w.key0 = keys.x;
                    w.keys = keys.y;
                    w.kv_head = unit / group;
                    const int tile = (unit - w.kv_head * group) * kTiles;
                    something = false;
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) {
                        const bool upper = tile + t >= group;
                        w.row0[t] = blk.row0 + (upper ? tokens : 0);
                        w.head[t] = (w.kv_head * group + tile + t - (upper ? group : 0)) * pack;
                        const int last = min(w.row0[t] + tokens, blk.rows) - 1, seen = a.causal ? min(last + keys.y - blk.rows + 1, keys.y) : keys.y;
                        w.n[t] = w.row0[t] >= blk.rows || seen <= 0 ? 0 : (seen + 127) / 128;
                        something |= w.row0[t] < blk.rows;
                    }
                }
                if (something) {                      // (numbers without a tile are passed over)
                    if ((threadIdx.x & 31) == 0) {
                        b->work = w;
                        ptx::mbar_arrive(&b->work_full);
                    }
                    // (a block is taken when the one before it is begun: taken earlier, it would wait here while other CTAs have none)
                    if (w.rows < 0 || !attn_wait_warp(&b->work_read, handed & 1, failed, a.report, 7)) break;
                    ++handed;
                }
                if ((threadIdx.x & 31) == 0) request_work(b);
                if (!attn_wait_warp(&b->answered, answers & 1, failed, a.report, 7)) break;
                item = work_of_answer(b);
                something = true;
                __syncwarp();
            }
        }
    } else {
        take_registers<Shape::kRegisters>();
        const int t = warp >> 2, lane_row = threadIdx.x & 127;
        const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16), ts = lanes + t * 128, to = lanes + Shape::kOut + t * 128;
        const float c = a.scale * kLog2e;
        uint32_t made = 0, ended = 0;                 // blocks of scores, of results so far
        const int token_of = lane_row / pack, head_of = lane_row - token_of * pack;
        FwdWork w;
        bool ok = true;
        for (int k = 0; ok && next_work(k, w); ++k) {
            const int row0 = t == 0 ? w.row0[0] : w.row0[1], head = (t == 0 ? w.head[0] : w.head[1]) + head_of, row = row0 + token_of, shift = w.keys - w.rows;
            const int seen = a.causal ? min(row + shift + 1, w.keys) : w.keys;      // keys that this row sees
            const int first_seen = a.causal ? min(row0 + shift + 1, w.keys) : w.keys;      // ... and the tile's first row
            const int n = t == 0 ? w.n[0] : w.n[1];
            float ref = 0.f, sum = 0.f;
            for (int j = 0; j < n; ++j) {
                ok = attn_wait_warp(&b->s_full[t], made & 1, failed, a.report, 5);
                if (!ok) break;
                ++made;
                umma::fence_after_thread_sync();
                uint32_t s[4][32];
                const bool masked = j * 128 + 128 > first_seen;
                const int visible = seen - j * 128;
                uint32_t out[32];
                uint64_t part[2];
                // 16 scores at a time, in an order that keeps the special function unit fed: scaled two steps ahead, summed and rounded a step behind
                auto scaled = [&](int i) {
                    const uint64_t c2 = f32x2(c, c), minus = f32x2(-ref * c, -ref * c);
#pragma unroll
                    for (int k = i * 16; k < i * 16 + 16; k += 2) {
                        float x, y;
                        umma::unpack_f32x2(fma2(umma::pack_f32x2(s[k >> 5][k & 31], s[k >> 5][(k & 31) + 1]), c2, minus), x, y);
                        s[k >> 5][k & 31] = __float_as_uint(x);
                        s[k >> 5][(k & 31) + 1] = __float_as_uint(y);
                    }
                };
                auto powers = [&](int i) {
#pragma unroll
                    for (int k = i * 16; k < i * 16 + 16; k += 2) {
                        uint32_t &x = s[k >> 5][k & 31], &y = s[k >> 5][(k & 31) + 1];
                        if ((k >> 1) % kPolynomialOf == kPolynomialOf - 1) {
                            float u, v;
                            umma::unpack_f32x2(exp2_by_polynomial(umma::pack_f32x2(x, y)), u, v);
                            x = __float_as_uint(u);
                            y = __float_as_uint(v);
                        } else {
                            x = __float_as_uint(exp2_approx(__uint_as_float(x)));
                            y = __float_as_uint(exp2_approx(__uint_as_float(y)));
                        }
                    }
                };
                auto rounded = [&](int i) {
#pragma unroll
                    for (int k = i * 16; k < i * 16 + 16; k += 2) {
                        const uint32_t x = s[k >> 5][k & 31], y = s[k >> 5][(k & 31) + 1];
                        part[(k >> 1) & 1] = add2(part[(k >> 1) & 1], umma::pack_f32x2(x, y));
                        out[(k & 63) >> 1] = pack_bf16(__uint_as_float(x), __uint_as_float(y));
                    }
                };
                auto hand_over = [&](int i) {
                    umma::tmem_st_32x32(ts + i * 32, out);
                    umma::tmem_st_wait();
                    umma::fence_before_thread_sync();
                    __syncwarp();
                    if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(&b->p_full[t][i]);
                };
#pragma unroll
                for (int i = 0; i < 4; ++i) umma::tmem_ld_32x32(ts + i * 32, s[i]);
                umma::tmem_ld_wait();
                if (masked)
#pragma unroll
                    for (int i = 0; i < 4; ++i) hide(s[i], first_bits(visible - i * 32));
                float top[8];                             // (many short chains)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    auto value = [&](int k) { return __uint_as_float(s[i >> 1][(i & 1) * 16 + k]); };
                    top[i] = max3(value(0), value(1), value(2));
#pragma unroll
                    for (int k = 3; k < 15; k += 2) top[i] = max3(top[i], value(k), value(k + 1));
                    top[i] = max3(top[i], value(15), value(15));
                }
                const float largest = max3(max3(max3(top[0], top[1], top[2]), top[3], top[4]), max3(top[5], top[6], top[7]), kNone);
                // The reference moves only when the largest score is more than 2^8 above it: sums and probabilities have that much room, and O is seldom multiplied.
                // With a score that is no number the reference is none either, and so are the row's sum, result and lse.
                if (j == 0) {
                    ref = largest == kNone ? 0.f : largest;
                } else {
                    const bool move = !((largest - ref) * c <= 8.f);
                    if (__any_sync(0xffffffffu, move)) {
                        const float factor = move ? exp2_approx((ref - largest) * c) : 1.f;
                        sum *= factor;
                        ref = move ? largest : ref;
#pragma unroll
                        for (int i = 0; i < 64 * kChunks; i += 16) {
                            uint32_t o[16];
                            umma::tmem_ld_32x16(to + i, o);
                            umma::tmem_ld_wait();
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * factor);
                            umma::tmem_st_32x16(to + i, o);
                        }
                    }
                }
                part[0] = f32x2(sum, 0.f);
                part[1] = f32x2(0.f, 0.f);
                scaled(0);
                scaled(1);
                powers(0);
#pragma unroll
                for (int i = 1; i < 8; ++i) {
                    if (i < 7) scaled(i + 1);
                    powers(i);
                    rounded(i - 1);
                    if (i == 4) hand_over(0);
                }
                rounded(7);
                hand_over(1);
                float u, v;
                umma::unpack_f32x2(add2(part[0], part[1]), u, v);
                sum = u + v;
            }
            const bool in = row < w.rows && token_of < tokens;
            const int64_t token = w.start + row;
            bf16* out = reinterpret_cast<bf16*>(a.o) + (token * a.heads + head) * a.dim;
            if (n > 0) {
                ok = ok && attn_wait_warp(&b->o_full[t], ended & 1, failed, a.report, 6);
                ++ended;
                if (ok) {
                    umma::fence_after_thread_sync();
                    store_row<64 * kChunks>(to, sum == 0.f ? 0.f : 1.f / sum, out, a.dim, in);
                }
            } else if (in) {
                for (int i = 0; i < a.dim; i += 8) *reinterpret_cast<uint4*>(out + i) = make_uint4(0, 0, 0, 0);
            }
            if (in && ok) a.lse[static_cast<int64_t>(head) * a.tq + token] = sum == 0.f ? kNone : (ref * c + log2f(sum)) * kLn2;
        }
    }
    umma::fence_before_thread_sync();
    __syncthreads();
    if (b->st.failed != 0) {
        // (a wait has run out: what was requested or issued ends before its memory goes to others)
        if (warp == Shape::kLoadWarp) {
            for (int i = 0; i < kTiles; ++i) mbar_drain(&b->q_full[i], 0, kLandNs), mbar_drain(&b->q_full[i], 1, kLandNs);
            for (int i = 0; i < kStages; ++i) mbar_drain(&b->full[i], 0, kLandNs), mbar_drain(&b->full[i], 1, kLandNs);
            mbar_drain(&b->answered, 0, kLandNs), mbar_drain(&b->answered, 1, kLandNs);
            mbar_drain(&b->tail, 0, kLandNs), mbar_drain(&b->tail, 1, kLandNs);
        }
        if (warp >= Shape::kMultiplyWarp && warp < Shape::kWorkWarp && ptx::elect_one()) {
            umma::mma_commit(&b->quiet[warp - Shape::kMultiplyWarp]);
            mbar_drain(&b->quiet[warp - Shape::kMultiplyWarp], 0, 1000000000ull);
        }
        __syncthreads();
    }
    if (warp == Shape::kMultiplyWarp) umma::tmem_dealloc(tmem, Shape::kColumns);
}

// ------------------------------------------------------------------------------------------------ backward
// delta = rowsum(dO O) - d_lse: 16 lanes per row of a head
constexpr int kDeltaThreads = 256;
__global__ void __launch_bounds__(kDeltaThreads) attention_delta_kernel(const __grid_constant__ AttentionArgs a) {
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * kDeltaThreads + threadIdx.x) / 16;
    const int lane = threadIdx.x & 15, c = lane * 8;
    const int64_t token = row / a.heads;
    const int head = static_cast<int>(row - token * a.heads);
    const bool in = token < a.tq;
    float sum = 0.f;
    if (in && c < a.dim) {
        const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const bf16*>(a.d_o.data) + token * a.d_o.stride_token + head * a.d_o.stride_head + c);
        const uint4 y = *reinterpret_cast<const uint4*>(static_cast<const bf16*>(a.o_in.data) + token * a.o_in.stride_token + head * a.o_in.stride_head + c);
        const uint32_t u[4] = {x.x, x.y, x.z, x.w}, v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sum = fmaf(__uint_as_float(u[i] << 16), __uint_as_float(v[i] << 16), sum);
            sum = fmaf(__uint_as_float(u[i] & 0xffff0000u), __uint_as_float(v[i] & 0xffff0000u), sum);
        }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (in && lane == 0) {
        const int64_t at = static_cast<int64_t>(head) * a.tq + token;
        a.delta[at] = a.d_lse != nullptr ? sum - a.d_lse[at] : sum;
    }
}

// A CTA keeps 128 rows of one side (kKeys: keys and values, whose gradients it makes; otherwise queries and dO, for dQ) and takes those of the other side in
// pieces of 128.  Scores and dP of a piece are products whose lanes are the kept rows, so that P and dS are first operands of the products that follow, and sums stay in
// tensor memory until the end: every gradient is added by one CTA (or by one per part of the group, whose parts are then added), in a fixed order.  P is made twice, which
// costs two products of seven, and spares sums of dQ in memory by many CTAs in any order.
//
// 16384 tokens, 56 heads of 128: 11.5 ms, 0.84 PFLOP/s counted as five products and 1.17 as seven, bound by power as the forward pass; two documents of 4096: 1.4 to 1.7 ms.  Short sequences are bound
// by the chain of a piece, some 2200 clocks, and by what a block takes to begin and to end.  There, too, tiles of queries take heads of a group together (31 x 264 tokens, 56 heads: 385 -> 280 to 291 us,
// 200 x 30, 32 heads: 324 -> 155).
//
// Two groups of four warps have 64 columns of a piece each.  P and dS take the place of dP; that of the scores is free as soon as they are in registers, so the next piece's
// scores are made meanwhile, and their powers while dV, dK and the next dP are.  (Pieces of 64 columns with two places for each had products of half the width, which take as long
// as whole ones: 128 rows of the first operand come from shared memory either way.)
constexpr int kBwdThreads = 384;                     // 2 x 4 warps for rows, one that requests pieces, one that issues products, one that looks for work, one without any
constexpr int kBwdReaders = 10;
template <int kChunks>
struct BwdShape {
    static constexpr int kTileBytes = 128 * 128 * kChunks, kSlots = kChunks == 2 ? 5 : 8;
    static constexpr int kStatBytes = 2 * 2 * 128 * 4;
    static constexpr int kSmem = (2 + kSlots) * kTileBytes + kStatBytes + 1024;
};
// Tensor memory of a block: sums (of keys and values, or of queries), scores, dP (once, or, of queries, in turn by pieces)
template <bool kKeys>
struct BwdColumns {
    static constexpr uint32_t kScores = kKeys ? 256 : 128;
    static __device__ __forceinline__ uint32_t dp(uint32_t piece) { return kKeys ? 384 : 256 + (piece & 1) * 128; }
};
struct BwdWork {
    int keys;                        // whether the block is one of keys
    int start, row0, rows;           // as of AttnBlock; rows < 0: no more work
    int other0, others;              // rows of the other side
    int head, first_head, split;     // (first) kept head, first head of the pieces
    int piece0, per_head, first, n;  // pieces [piece0, piece0 + per_head) of every head (or of `pack` at once); of all of them n from `first` on
    // the head and the piece of the i-th
    __device__ __forceinline__ int head_of(int i, int pack) const { return first_head + (first + i) / per_head * pack; }
    __device__ __forceinline__ int piece_of(int i) const { return piece0 + (first + i) % per_head; }
};
// (dP and what is made of it in turn by pieces: with two places for dP, the next one's can be there before a slow warp has looked for this one's)
struct BwdBars {
    alignas(16) uint4 answer;
    BwdWork work;
    uint64_t kept, kept_empty, full[8], empty[8], s_full, s_read, dp_full[2], p_full[2][2], stats_full[2], sums, drained, work_full, work_read, answered, tail, quiet;
    AttnState st;
};
static_assert(sizeof(BwdBars) <= 1024, "what BwdShape leaves for it");

// Blocks of keys and blocks of queries are one launch, those of keys first: a CTA takes either as they come, so that the SMs which the last keys leave free go on with queries (1000 tokens of 8
// heads of 128: 25 us, with a launch for each 40; two documents of 4096, 56 heads: 1420 to 1470, 1640 to 1670).  Both read delta, which the kernel before this one makes, and nothing that the other makes.
template <int kChunks>
__global__ void __launch_bounds__(kBwdThreads, 1)
attention_backward_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_q,
                          const __grid_constant__ CUtensorMap map_d, const __grid_constant__ AttentionArgs a) {
    using Shape = BwdShape<kChunks>;
    using Keys = std::true_type;
    using Queries = std::false_type;
    constexpr int kSlots = Shape::kSlots, kTileBytes = Shape::kTileBytes;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *kept = smem, *pieces = smem + 2 * kTileBytes;
    float* stats = reinterpret_cast<float*>(pieces + kSlots * kTileBytes);
    BwdBars* b = reinterpret_cast<BwdBars*>(pieces + kSlots * kTileBytes + Shape::kStatBytes);
    const int warp = threadIdx.x >> 5, group = a.heads / a.kv_heads;
    // queries lie in tiles of `tokens` times `pack` heads, keys in tiles of 128
    const int pack = a.pack, tokens = 128 / pack;
    if (threadIdx.x == 0) {
        umma::prefetch_tensormap(&map_k);
        umma::prefetch_tensormap(&map_v);
        umma::prefetch_tensormap(&map_q);
        umma::prefetch_tensormap(&map_d);
        ptx::mbar_init(&b->kept, 1);
        ptx::mbar_init(&b->kept_empty, 1);
        ptx::mbar_init(&b->drained, 8);
        ptx::mbar_init(&b->work_full, 1);
        ptx::mbar_init(&b->work_read, kBwdReaders);
        ptx::mbar_init(&b->answered, 1);
        for (int i = 0; i < kSlots; ++i) {
            ptx::mbar_init(&b->full[i], 1);
            ptx::mbar_init(&b->empty[i], 1);
        }
        ptx::mbar_init(&b->s_full, 1);
        ptx::mbar_init(&b->s_read, 8);
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&b->dp_full[i], 1);
            ptx::mbar_init(&b->p_full[i][0], 4);
            ptx::mbar_init(&b->p_full[i][1], 4);
            ptx::mbar_init(&b->stats_full[i], 4);
        }
        ptx::mbar_init(&b->sums, 1);
        ptx::mbar_init(&b->tail, 1);
        ptx::mbar_init(&b->quiet, 1);
        b->st.failed = 0;
        ptx::mbar_fence_init();
    }
    if (warp == 9) {
        umma::tmem_alloc(&b->st.tmem_base, 512);
        umma::tmem_relinquish();
    }
    if (warp == 8) {                                     // (rows that no query has)
        for (int i = 0; i < 2 + kSlots; ++i) clear_tile<128, kChunks>(smem + i * kTileBytes, tokens * pack);
    }
    umma::fence_before_thread_sync();
    __syncthreads();
    umma::fence_after_thread_sync();
    const uint32_t tmem = b->st.tmem_base;
    ptx::wait_for_previous_kernel();
    int* failed = &b->st.failed;
    // The k-th block of this CTA, for a whole warp; false: no more
    auto next_work = [&](int k, BwdWork& w) {
        if (!attn_wait_warp(&b->work_full, k & 1, failed, a.report, 7)) return false;
        w = b->work;
        __syncwarp();
        if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(&b->work_read);
        return w.rows >= 0;
    };

    if (warp >= 8) {
        give_registers<3 * 168 - 2 * kBwdRegisters>();
        if (warp == 8) {
            AttnRing<kSlots> p;
            const bool one = ptx::elect_one();
            uint32_t tails = 0, blocks = 0, whole = 0;   // whole: stages (bits) whose last tile was one of keys, with rows that no query has
            auto request = [&](auto kind, const BwdWork& w, const CUtensorMap* map, int h, int piece) {
                constexpr bool kKeys = decltype(kind)::value;
                const int step = kKeys ? tokens : 128;
                if (!attn_wait_warp(&b->empty[p.stage], p.phase ^ 1, failed, a.report, 1)) return false;
                uint8_t* tile = pieces + p.stage * kTileBytes;
                if (!kKeys) {
                    whole |= 1u << p.stage;
                } else if (whole >> p.stage & 1u) {
                    clear_tile<128, kChunks>(tile, tokens * pack);
                    whole &= ~(1u << p.stage);
                }
                const bool tail = piece * step + step > w.others;
                uint64_t* bar = tail ? &b->tail : &b->full[p.stage];
                if (one) {
                    ptx::mbar_arrive_expect_tx(bar, kKeys ? tokens * pack * 128 * kChunks : kTileBytes);
                    load_tile<128, kChunks>(tile, map, h, w.other0 + piece * step, bar);
                }
                __syncwarp();
                if (tail) {
                    if (!attn_wait_warp(&b->tail, tails & 1, failed, a.report, 4)) return false;
                    ++tails;
                    clear_tile<128, kChunks>(tile, (w.others - piece * step) * (kKeys ? pack : 1));
                    if (one) ptx::mbar_arrive(&b->full[p.stage]);
                }
                p.advance();
                return true;
            };
            auto load = [&](auto kind, const BwdWork& w) {
                constexpr bool kKeys = decltype(kind)::value;
                if (w.n == 0) return true;
                if (!attn_wait_warp(&b->kept_empty, (blocks & 1) ^ 1, failed, a.report, 1)) return false;
                ++blocks;
                if (one) {
                    ptx::mbar_arrive_expect_tx(&b->kept, 2 * (kKeys ? kTileBytes : tokens * pack * 128 * kChunks));
                    load_tile<128, kChunks>(kept, kKeys ? &map_k : &map_q, w.head, w.start + w.row0, &b->kept);
                    load_tile<128, kChunks>(kept + kTileBytes, kKeys ? &map_v : &map_d, w.head, w.start + w.row0, &b->kept);
                }
                __syncwarp();
                for (int i = 0; i < w.n; ++i) {
                    const int h = kKeys ? w.head_of(i, pack) : w.head / group, piece = w.piece_of(i);
                    if (!request(kind, w, kKeys ? &map_q : &map_k, h, piece) || !request(kind, w, kKeys ? &map_d : &map_v, h, piece)) return false;
                }
                return true;
            };
            BwdWork w;
            for (int k = 0; next_work(k, w); ++k)
                if (!(w.keys ? load(Keys{}, w) : load(Queries{}, w))) break;
        } else if (warp == 9) {
            const bool one = ptx::elect_one();
            const int dim16 = (a.dim + 15) / 16;
            const uint32_t idesc_s = umma::make_instr_desc(128, 128, umma::kFormatBF16);
            const uint32_t idesc_o = umma::make_instr_desc(128, 16, umma::kFormatBF16, false, true) + (static_cast<uint32_t>(2 * dim16 - 2) << 17);
            const uint32_t kept_of = desc_channels(kept), pieces_of = desc_channels(pieces), rows_of = desc_rows<128>(pieces);
            AttnRing<kSlots> p;                       // operands in the order in which they come: first and second of every piece
            uint32_t made = 0, blocks = 0;            // pieces, blocks so far
            int keys_before = 0;                      // kind of the block before
            // the first products of a piece, of its first or second operand
            auto product = [&](int which, uint32_t to, uint64_t* done, int& slot) {
                if (!attn_wait(&b->full[p.stage], p.phase, failed, a.report, 4)) return false;
                umma::fence_after_thread_sync();
                multiply_channels<128, 128, kChunks>(tmem + to, kept_of + which * (kTileBytes / 16), pieces_of + p.stage * (kTileBytes / 16), idesc_s, dim16);
                umma::mma_commit(done);
                slot = p.stage;
                p.advance();
                return true;
            };
            auto multiply = [&](auto kind, int n) {
                constexpr bool kKeys = decltype(kind)::value;
                using Columns = BwdColumns<kKeys>;
                // (the sums of the block before have been read: of another kind, they lie where this one's first products go)
                if (blocks > 0 && keys_before != kKeys && !attn_wait(&b->drained, (blocks - 1) & 1, failed, a.report, 6)) return;
                keys_before = kKeys;
                if (!attn_wait(&b->kept, blocks & 1, failed, a.report, 4)) return;
                int slot0, slot1, next0 = 0, next1 = 0;
                if (!product(0, Columns::kScores, &b->s_full, slot0) || !product(1, Columns::dp(made), &b->dp_full[made & 1], slot1)) return;
                if (!kKeys) umma::mma_commit(&b->empty[slot1]);
                if (n == 1) umma::mma_commit(&b->kept_empty);
                if (blocks > 0 && !attn_wait(&b->drained, (blocks - 1) & 1, failed, a.report, 6)) return;
                ++blocks;
                for (int i = 0; i < n; ++i, ++made) {
                    const uint32_t dp = Columns::dp(made);
                    if (i + 1 < n) {
                        if (!attn_wait(&b->s_read, made & 1, failed, a.report, 3)) return;
                        if (!product(0, Columns::kScores, &b->s_full, next0)) return;
                        if (!kKeys) {
                            // (the other place of dP: what was there is behind the products before)
                            if (!product(1, Columns::dp(made + 1), &b->dp_full[~made & 1], next1)) return;
                            umma::mma_commit(&b->empty[next1]);
                            if (i + 2 == n) umma::mma_commit(&b->kept_empty);
                        }
                    }
                    const uint32_t rows0 = rows_of + slot0 * (kTileBytes / 16), rows1 = rows_of + slot1 * (kTileBytes / 16);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if (!attn_wait(&b->p_full[half][made & 1], made >> 1 & 1, failed, a.report, 2)) return;
                        umma::fence_after_thread_sync();
                        const uint32_t from = tmem + dp + half * 64, step = half * 4 * 16 * 128 / 16;
                        if (kKeys) multiply_rows<0, 4>(tmem + 128, from, rows1 + step, idesc_o, i != 0 || half != 0);
                        multiply_rows<0, 4>(tmem, from + 32, rows0 + step, idesc_o, i != 0 || half != 0);
                    }
                    umma::mma_commit(&b->empty[slot0]);
                    if (kKeys) {
                        umma::mma_commit(&b->empty[slot1]);
                        if (i + 1 < n) {
                            if (!product(1, Columns::dp(made + 1), &b->dp_full[~made & 1], next1)) return;
                            if (i + 2 == n) umma::mma_commit(&b->kept_empty);
                        }
                    }
                    slot0 = next0;
                    slot1 = next1;
                }
                umma::mma_commit(&b->sums);
                // (nobody waits for the last piece's scores to be read)
            };
            BwdWork w;
            for (int k = 0; next_work(k, w); ++k) {
                if (one && w.n > 0) {
                    if (w.keys) multiply(Keys{}, w.n);
                    else multiply(Queries{}, w.n);
                }
                __syncwarp();
            }
        } else if (warp == 10) {
            // looks for work: first this CTA's own
            int item = blockIdx.x;
            uint32_t handed = 0;
            for (uint32_t answers = 0;; ++answers) {
                BwdWork w{};
                w.rows = -1;
                bool something = true;
                if (item >= 0) {
                    // (keys: the first ones are seen by most queries; queries: the last ones see most keys.  Long blocks first.)
                    const bool keys = item < a.key_ctas;
                    const int units = keys ? a.kv_heads * a.splits : a.heads / pack, mine = keys ? item : item - a.key_ctas, all_mine = keys ? a.key_ctas : gridDim.x - a.key_ctas;
                    const int unit = mine % units, number = mine / units, step = keys ? tokens : 128;
                    w.keys = keys;
                    w.head = keys ? unit / a.splits : unit * pack;      // (of keys, or of queries)
                    w.split = keys ? unit % a.splits : 0;
                    w.first_head = keys ? w.head * group : 0;
                    const AttnBlock blk = find_block(keys ? a.cu_k : a.cu_q, a.num_seqs, keys ? a.tk : a.tq, keys ? number : all_mine / units - 1 - number, keys ? 128 : tokens);
                    const int2 other = sequence_rows(keys ? a.cu_q : a.cu_k, blk.seq, keys ? a.tq : a.tk);
                    const int shift = keys ? blk.rows - other.y : other.y - blk.rows;
                    w.start = blk.start;
                    w.row0 = blk.row0;
                    w.rows = blk.rows;
                    w.other0 = other.x;
                    w.others = other.y;
                    something = blk.row0 < blk.rows;
                    int piece1 = (other.y + step - 1) / step;
                    if (keys) {
                        w.piece0 = a.causal ? max(blk.row0 - shift, 0) / step : 0;
                    } else if (a.causal) {
                        const int seen = min(min(blk.row0 + tokens, blk.rows) + shift, other.y);
                        piece1 = seen <= 0 ? 0 : (seen + 127) / 128;
                    }
                    w.per_head = max(piece1 - w.piece0, 0);
                    // (a part of the group's pieces, of all heads)
                    const int64_t all = static_cast<int64_t>(w.per_head) * (keys ? group / pack : 1);
                    w.first = static_cast<int>(keys ? all * w.split / a.splits : 0);
                    w.n = static_cast<int>((keys ? all * (w.split + 1) / a.splits : all) - w.first);
                    const int64_t row_values = static_cast<int64_t>(keys ? a.kv_heads : a.heads) * a.dim;
                    if (!keys) {
                        clear_rows<32>(a.cu_q, a.num_seqs, a.tq, mine, all_mine, reinterpret_cast<bf16*>(a.dq), row_values, nullptr, 0);
                    } else if (a.splits == 1) {
                        clear_rows<32>(a.cu_k, a.num_seqs, a.tk, mine, all_mine, reinterpret_cast<bf16*>(a.dk), row_values, nullptr, 0);
                        clear_rows<32>(a.cu_k, a.num_seqs, a.tk, mine, all_mine, reinterpret_cast<bf16*>(a.dv), row_values, nullptr, 0);
                    }
                }
                if (something) {                      // (numbers without a block are passed over)
                    if ((threadIdx.x & 31) == 0) {
                        b->work = w;
                        ptx::mbar_arrive(&b->work_full);
                    }
                    if (w.rows < 0 || !attn_wait_warp(&b->work_read, handed & 1, failed, a.report, 7)) break;
                    ++handed;
                }
                if ((threadIdx.x & 31) == 0) request_work(b);
                if (!attn_wait_warp(&b->answered, answers & 1, failed, a.report, 7)) break;
                item = work_of_answer(b);
                __syncwarp();
            }
        }
    } else {
        take_registers<kBwdRegisters>();
        const int half = warp >> 2, lane_row = threadIdx.x & 127;
        const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const float c = a.scale * kLog2e;
        float* stats_of_half = stats + half * 256;    // twice: 64 times -lse log2 e, 64 times -delta
        const uint64_t c2 = f32x2(c, c);
        uint32_t made = 0, told = 0, ended = 0;       // pieces, pieces with statistics, blocks so far
        // A block; false: a wait has run out
        auto rows = [&](auto kind, const BwdWork& w) {
            constexpr bool kKeys = decltype(kind)::value;
            using Columns = BwdColumns<kKeys>;
            const int step = kKeys ? tokens : 128;
            const int column = kKeys ? half * 64 + (lane_row & 63) : lane_row, token_of = column / pack, head_of = column - token_of * pack;      // of what this thread reads statistics of
            const int row = w.row0 + (kKeys ? lane_row : token_of), shift = kKeys ? w.rows - w.others : w.others - w.rows;     // query i sees the keys up to i + shift
            const bool in = row < w.rows && (kKeys || token_of < tokens);
            const int64_t token = w.start + row;
            const int head = w.head + (kKeys ? 0 : head_of);
            // a statistic of a query that sees nothing, or that is none: its probabilities are zero
            auto statistic = [&](bool is_delta, bool is_there, int h, int64_t query) {
                if (!is_there) return is_delta ? 0.f : kNone;
                const int64_t at = static_cast<int64_t>(h) * a.tq + query;
                if (is_delta) return -a.delta[at];
                const float l = a.lse_in[at];
                return l == kNone ? kNone : -l * kLog2e;
            };
            auto next_statistic = [&](int i) {
                if (i >= w.n) return 0.f;
                const int at = w.piece_of(i) * tokens + token_of;
                return statistic(lane_row >= 64, token_of < tokens && at < w.others, w.head_of(i, pack) + head_of, w.other0 + at);
            };
            float coming = 0.f;
            uint64_t minus2 = 0, delta2 = 0;
            if (kKeys) {
                coming = next_statistic(0);
            } else if (w.n > 0) {
                const float m = statistic(false, in, head, token), d = statistic(true, in, head, token);
                minus2 = f32x2(m, m);
                delta2 = f32x2(d, d);
            }
            for (int i = 0; i < w.n; ++i, ++made) {
                float* now = stats_of_half + (told & 1) * 128;
                if (kKeys) {
                    now[lane_row] = coming;
                    __syncwarp();
                    if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(&b->stats_full[half]);
                    coming = next_statistic(i + 1);
                    if (!attn_wait_warp(&b->stats_full[half], told & 1, failed, a.report, 6)) return false;
                    ++told;
                }
                if (!attn_wait_warp(&b->s_full, made & 1, failed, a.report, 5)) return false;
                umma::fence_after_thread_sync();
                uint32_t s[2][32], d[2][32];
                umma::tmem_ld_32x32(lanes + Columns::kScores + half * 64, s[0]);
                umma::tmem_ld_32x32(lanes + Columns::kScores + half * 64 + 32, s[1]);
                umma::tmem_ld_wait();
                umma::fence_before_thread_sync();
                __syncwarp();
                if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(&b->s_read);
                const int first = w.piece_of(i) * step;
                // columns [low, high) are visible
                int low = 0, high = 64;
                if (kKeys) {
                    if (a.causal) low = min(max(row - shift - first, 0), tokens) * pack - half * 64;
                } else {
                    high = (a.causal ? min(row + shift + 1, w.others) : w.others) - first - half * 64;
                }
                const bool masked = __any_sync(0xffffffffu, low > 0 || high < 64);
#pragma unroll
                for (int k = 0; k < 64; k += 2) {
                    if (kKeys) {
                        const float2 m = *reinterpret_cast<const float2*>(now + k);
                        minus2 = f32x2(m.x, m.y);
                    }
                    float x, y;
                    umma::unpack_f32x2(fma2(umma::pack_f32x2(s[k >> 5][k & 31], s[k >> 5][(k & 31) + 1]), c2, minus2), x, y);
                    s[k >> 5][k & 31] = __float_as_uint(x);
                    s[k >> 5][(k & 31) + 1] = __float_as_uint(y);
                }
                if (masked)
#pragma unroll
                    for (int k = 0; k < 64; ++k)
                        if (k < low || k >= high) s[k >> 5][k & 31] = 0xff800000u;
#pragma unroll
                for (int k = 0; k < 64; ++k) s[k >> 5][k & 31] = __float_as_uint(exp2_approx(__uint_as_float(s[k >> 5][k & 31])));
                if (!attn_wait_warp(&b->dp_full[made & 1], made >> 1 & 1, failed, a.report, 5)) return false;
                umma::fence_after_thread_sync();
                const uint32_t dp = lanes + Columns::dp(made) + half * 64;
                umma::tmem_ld_32x32(dp, d[0]);
                umma::tmem_ld_32x32(dp + 32, d[1]);
                umma::tmem_ld_wait();
                uint32_t out[32];
                if (kKeys) {
#pragma unroll
                    for (int k = 0; k < 64; k += 2) out[k >> 1] = pack_bf16(__uint_as_float(s[k >> 5][k & 31]), __uint_as_float(s[k >> 5][(k & 31) + 1]));
                    umma::tmem_st_32x32(dp, out);
                }
#pragma unroll
                for (int k = 0; k < 64; k += 2) {
                    if (kKeys) {
                        const float2 m = *reinterpret_cast<const float2*>(now + 64 + k);
                        delta2 = f32x2(m.x, m.y);
                    }
                    float u, v;
                    umma::unpack_f32x2(mul2(umma::pack_f32x2(s[k >> 5][k & 31], s[k >> 5][(k & 31) + 1]), add2(umma::pack_f32x2(d[k >> 5][k & 31], d[k >> 5][(k & 31) + 1]), delta2)), u, v);
                    out[k >> 1] = pack_bf16(u, v);
                }
                if (masked) {                             // (zero whatever dP is there)
#pragma unroll
                    for (int k = 0; k < 64; k += 2) {
                        const uint32_t keep = (k >= low && k < high ? 0xffffu : 0u) | (k + 1 >= low && k + 1 < high ? 0xffff0000u : 0u);
                        out[k >> 1] &= keep;
                    }
                }
                umma::tmem_st_32x32(dp + 32, out);
                umma::tmem_st_wait();
                umma::fence_before_thread_sync();
                __syncwarp();
                if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(&b->p_full[half][made & 1]);
            }
            const int64_t at = (token * (kKeys ? a.kv_heads : a.heads) + head) * a.dim;
            const float factor = kKeys && half == 1 ? 1.f : a.scale;
            bf16* out = reinterpret_cast<bf16*>(kKeys ? (half == 0 ? a.dk : a.dv) : a.dq) + at;
            float* part = nullptr;
            if (kKeys && a.splits > 1) part = a.parts + (static_cast<int64_t>(w.split) * 2 + half) * a.tk * a.kv_heads * a.dim + at;
            if (w.n > 0) {
                if (!attn_wait_warp(&b->sums, ended & 1, failed, a.report, 6)) return false;
                ++ended;
                umma::fence_after_thread_sync();
                if (!kKeys) {
                    const int first = half * 32 * kChunks;
                    store_row<32 * kChunks>(lanes + first, factor, out + first, a.dim - first, in);
                } else if (part != nullptr) {
                    store_part<64 * kChunks>(lanes + half * 128, factor, part, a.dim, in);
                } else {
                    store_row<64 * kChunks>(lanes + half * 128, factor, out, a.dim, in);
                }
                umma::fence_before_thread_sync();
                __syncwarp();
                if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(&b->drained);
            } else if (in && (kKeys || half == 0)) {
                for (int i = 0; i < a.dim; i += 8) {
                    if (part != nullptr) *reinterpret_cast<uint4*>(part + i) = *reinterpret_cast<uint4*>(part + i + 4) = make_uint4(0, 0, 0, 0);
                    else *reinterpret_cast<uint4*>(out + i) = make_uint4(0, 0, 0, 0);
                }
            }
            return true;
        };
        BwdWork w;
        for (int k = 0; next_work(k, w); ++k)
            if (!(w.keys ? rows(Keys{}, w) : rows(Queries{}, w))) break;
    }
    umma::fence_before_thread_sync();
    __syncthreads();
    if (b->st.failed != 0) {
        // (as in the forward pass)
        if (warp == 8) {
            mbar_drain(&b->kept, 0, kLandNs), mbar_drain(&b->kept, 1, kLandNs);
            mbar_drain(&b->answered, 0, kLandNs), mbar_drain(&b->answered, 1, kLandNs);
            mbar_drain(&b->tail, 0, kLandNs), mbar_drain(&b->tail, 1, kLandNs);
            for (int i = 0; i < kSlots; ++i) mbar_drain(&b->full[i], 0, kLandNs), mbar_drain(&b->full[i], 1, kLandNs);
        }
        if (warp == 9 && ptx::elect_one()) {
            umma::mma_commit(&b->quiet);
            mbar_drain(&b->quiet, 0, 1000000000ull);
        }
        __syncthreads();
    }
    if (warp == 9) umma::tmem_dealloc(tmem, 512);
}

// The parts of dK and dV, in their order; rows of no sequence get zeros
constexpr int kAddThreads = 256;
__global__ void __launch_bounds__(kAddThreads) attention_add_kernel(const __grid_constant__ AttentionArgs a) {
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const int64_t row_values = static_cast<int64_t>(a.kv_heads) * a.dim, values = a.tk * row_values;
    const int64_t at = (static_cast<int64_t>(blockIdx.x) * kAddThreads + threadIdx.x) * 4;
    if (at >= values) return;
    const int row = static_cast<int>(at / row_values), first = a.cu_k == nullptr ? 0 : a.cu_k[0], last = a.cu_k == nullptr ? a.tk : a.cu_k[a.num_seqs];
    const bool in = row >= first && row < last;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        if (in)
#pragma unroll 4
            for (int i = 0; i < a.splits; ++i) {
                const float4 x = *reinterpret_cast<const float4*>(a.parts + (static_cast<int64_t>(i) * 2 + which) * values + at);
                sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
            }
        *reinterpret_cast<uint2*>(static_cast<bf16*>(which == 0 ? a.dk : a.dv) + at) = make_uint2(pack_bf16(sum.x, sum.y), pack_bf16(sum.z, sum.w));
    }
}

// ------------------------------------------------------------------------------------------------ host
bool make_map(CUtensorMap* map, const HeadsView& x, int64_t tokens, int64_t heads, int64_t dim, int box_rows, int box_heads = 1) {
    EncodeTiledFn encode = get_encode_fn();
    if (encode == nullptr) return false;
    // (a stride that nothing steps along may be anything)
    const int64_t pitch = (dim * 2 + 15) / 16 * 16;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(heads > 1 ? x.stride_head * 2 : pitch), static_cast<cuuint64_t>(tokens > 1 ? x.stride_token * 2 : pitch)};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t steps[3] = {1, 1, 1};
    auto made = [&]() {
        return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(x.data), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    if (made()) return true;
    // (the driver wants a context, and a thread that has made no call of the runtime yet, as those that run gradients, has none)
    int device = 0;
    return cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess && made();
}
// leave for shared memory, once per device
cudaError_t allow_once(const void* fn, int bytes, std::atomic<uint64_t>& allowed) {
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) return err;
    if (device >= 64 || (allowed.load(std::memory_order_relaxed) >> device & 1) == 0) {
        err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (err != cudaSuccess) cudaGetLastError();      // the caller reports it
        else if (device < 64) allowed.fetch_or(1ull << device, std::memory_order_relaxed);
    }
    return err;
}

// Small tasks are sequences of so many keys or fewer on average, or few tiles for the SMs: tiles of queries take heads together, and the forward pass one tile per CTA.  Forward: 8 x 1000 tokens of 56
// heads 150 instead of 157 us, 8 x 1500 of 32 heads 196 instead of 221, 8 x 2000 of 56 485 instead of 471; one of 4096 with 16 heads (512 tiles) 81 instead of 97, with 32 (1024) 126 instead of 131, with 56
// (1792) 223 instead of 213, one of 8192 with 16 (1024) 234 instead of 229.  The average decides: a long prompt beside many short ones goes the way of the short ones.  Gradients (heads together or not): 16 x 450 285 instead of 320, 8 x 1500 598 instead of 620 to 637.
constexpr int kShortKeys = 2048, kFewTiles = 6;      // (tiles: per SM)
bool is_small(const AttentionArgs& a) {
    return a.tk / std::max(a.num_seqs, 1) <= kShortKeys || static_cast<int64_t>(a.tq) * a.heads / 128 < static_cast<int64_t>(kFewTiles) * a.num_sms;
}
// Heads that a tile takes of as many tokens as fill it: all of a group, or as many as divide it
int packed_heads(const AttentionArgs& a) {
    const int group = a.heads / a.kv_heads;
    int pack = std::min(group, kPackedHeads);
    while (group % pack != 0) --pack;
    return pack;
}
template <int kChunks, int kTiles>
cudaError_t launch_forward(AttentionArgs a, cudaStream_t stream) {
    using Shape = FwdShape<kChunks, kTiles>;
    const void* fn = reinterpret_cast<const void*>(attention_kernel<kChunks, kTiles>);
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t err = allow_once(fn, Shape::kSmem, allowed);
    if (err != cudaSuccess) return err;
    a.pack = is_small(a) ? packed_heads(a) : 1;
    const int tokens = 128 / a.pack;
    CUtensorMap q, k, v;
    if (!make_map(&q, a.q, a.tq, a.heads, a.dim, tokens, a.pack) || !make_map(&k, a.k, a.tk, a.kv_heads, a.dim, 128) || !make_map(&v, a.v, a.tk, a.kv_heads, a.dim, 128))
        return cudaErrorInvalidValue;
    void* params[] = {&q, &k, &v, &a};
    return launch_dependent(fn, dim3(static_cast<unsigned>(num_blocks(a.tq, a.num_seqs, kTiles * tokens) * (a.heads / a.pack))), dim3(Shape::kThreads), params, Shape::kSmem, stream);
}
template <int kChunks>
cudaError_t launch_forward(const AttentionArgs& a, cudaStream_t stream) {
    return is_small(a) ? launch_forward<kChunks, 1>(a, stream) : launch_forward<kChunks, 2>(a, stream);
}
template <int kChunks>
cudaError_t launch_backward(AttentionArgs a, cudaStream_t stream) {
    CUtensorMap q, k, v, d;
    a.pack = is_small(a) ? packed_heads(a) : 1;
    if (!make_map(&q, a.q, a.tq, a.heads, a.dim, 128 / a.pack, a.pack) || !make_map(&d, a.d_o, a.tq, a.heads, a.dim, 128 / a.pack, a.pack) || !make_map(&k, a.k, a.tk, a.kv_heads, a.dim, 128) ||
        !make_map(&v, a.v, a.tk, a.kv_heads, a.dim, 128))
        return cudaErrorInvalidValue;
    const void* fn = reinterpret_cast<const void*>(attention_backward_kernel<kChunks>);
    static std::atomic<uint64_t> allowed{0};
    cudaError_t err = allow_once(fn, BwdShape<kChunks>::kSmem, allowed);
    if (err != cudaSuccess) return err;
    const int64_t key_ctas = num_blocks(a.tk, a.num_seqs, 128) * a.kv_heads * a.splits, ctas = key_ctas + num_blocks(a.tq, a.num_seqs, 128 / a.pack) * (a.heads / a.pack);
    a.key_ctas = static_cast<int>(key_ctas);
    void *params[] = {&a}, *maps_and_args[] = {&k, &v, &q, &d, &a};
    const int64_t rows = static_cast<int64_t>(a.tq) * a.heads;
    err = launch_dependent(reinterpret_cast<const void*>(attention_delta_kernel), dim3(static_cast<unsigned>((rows * 16 + kDeltaThreads - 1) / kDeltaThreads)), dim3(kDeltaThreads), params, 0,
                           stream);
    if (err == cudaSuccess) err = launch_dependent(fn, dim3(static_cast<unsigned>(ctas)), dim3(kBwdThreads), maps_and_args, BwdShape<kChunks>::kSmem, stream);
    if (err == cudaSuccess && a.splits > 1) {
        const int64_t values = static_cast<int64_t>(a.tk) * a.kv_heads * a.dim;
        err = launch_dependent(reinterpret_cast<const void*>(attention_add_kernel), dim3(static_cast<unsigned>((values / 4 + kAddThreads - 1) / kAddThreads)), dim3(kAddThreads), params, 0,
                               stream);
    }
    return err;
}

}  // namespace

cudaError_t launch_attention(const AttentionArgs& a, cudaStream_t stream) {
    return a.dim <= 64 ? launch_forward<1>(a, stream) : launch_forward<2>(a, stream);
}
// Parts of a group whose gradients of keys and values are made by CTAs of their own, and then added (8 bytes per part and value each way): as many as give every SM two.
int attention_backward_splits(const AttentionArgs& a) {
    const int64_t ctas = std::max<int64_t>(1, std::max(a.tk / 128, 1) * a.kv_heads);
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(a.heads / a.kv_heads, 2 * a.num_sms / ctas)));
}
cudaError_t launch_attention_backward(const AttentionArgs& a, cudaStream_t stream) {
    return a.dim <= 64 ? launch_backward<1>(a, stream) : launch_backward<2>(a, stream);
}

}  // namespace ep
