// Attention of one new token per sequence over a paged cache:  o = softmax(scale q K^T) V  per query head, with the keys and values of its group's head, the first
// lengths[i] places of the sequence, place p in page page_table[i, p / page_size].
//
// Bound by memory: every key and value is read once for 16 query heads of a group (once more for every further 16 that a group has), 4 D bytes for 4 D operations per query head.
// A pair is a sequence and 16 query heads of a key head.  The pairs' keys are cut into tiles, 16 keys for each of a CTA's warps (one where pairs are many, otherwise four), in
// one line, and every CTA takes an equal stretch of it, whatever the lengths; a pair whose tiles lie with several CTAs is joined by a second kernel.  Where no sequence can have
// more than 512 keys a CTA takes a pair, and nothing is joined.  A warp has its own ring of asynchronous copies in shared memory and its own softmax in registers, so that no
// warp waits for another before a pair's end.
// Products are 16 x 8 x 16 (mma.sync): up to 16 query heads of a group are the rows, a thousandth of the tensor cores' rate, which is not what this waits for.
// Statistics and sums are 32 bits, probabilities are rounded to bf16 as operands.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"

namespace ep {

namespace {

using bf16 = __nv_bfloat16;
constexpr int kHeadRows = 16, kPagedStages = 3;
constexpr int kManyPairs = 2;                        // per SM
constexpr int kPairKeys = 512;                       // what a CTA takes of a pair where none has more
constexpr float kPagedLog2e = 1.4426950408889634f;
constexpr float kLowest = -__builtin_huge_valf();

// kWarps of a CTA share a tile, 16 keys each.  As many CTAs as the shared memory of an SM holds
template <int kDim, int kWarps>
struct PagedShape {
    static constexpr int kThreads = kWarps * 32, kTileKeys = kWarps * 16, kCtas = (kDim == 128 ? 8 : 16) / kWarps;
    static constexpr int kRowBytes = kDim * 2, kStageBytes = 2 * 16 * kRowBytes, kWarpBytes = kPagedStages * kStageBytes;
    static constexpr int kRing = kWarps * kWarpBytes;
    static constexpr int kPartFloats = kHeadRows * kDim + 2 * kHeadRows;      // sums, references, totals
    static_assert(kWarps * kHeadRows * kDim * 4 <= kRing, "the warps' sums lie in the ring");
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t v;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
    return v;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {      // zeros where nothing is
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void matrices(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void matrices_transposed(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ------------------------------------------------------------------------------------------------ the line of tiles
__device__ __forceinline__ int64_t capacity(const PagedAttentionArgs& a) { return static_cast<int64_t>(a.table_width) * a.page_size; }
__device__ __forceinline__ int keys_of(const PagedAttentionArgs& a, int seq) {      // (what the table cannot hold is not looked for: the result is no number)
    const int64_t n = a.lengths[seq];
    return static_cast<int>(max(static_cast<int64_t>(0), min(n, capacity(a))));
}
template <int kTileKeys>
__host__ __device__ __forceinline__ int tiles_of_keys(int keys) {
    return (keys + kTileKeys - 1) / kTileKeys;
}
// Every thread of a CTA of kThreads: first[i] = tiles in front of sequence i (of one key head), first[num_seqs] = all
template <int kThreads, int kTileKeys>
__device__ __forceinline__ void count_tiles(const PagedAttentionArgs& a, int* first) {
    __shared__ int s_warp[kThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int before = 0;
    for (int base = 0; base < a.num_seqs; base += kThreads) {
        const int i = base + threadIdx.x;
        const int n = i < a.num_seqs ? tiles_of_keys<kTileKeys>(keys_of(a, i)) : 0;
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 31) s_warp[warp] = upto;
        __syncthreads();
        int total = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) upto += s_warp[w];
            total += s_warp[w];
        }
        if (i < a.num_seqs) first[i] = before + upto - n;
        before += total;
        __syncthreads();
    }
    if (threadIdx.x == 0) first[a.num_seqs] = before;
    __syncthreads();
}
struct Stretch {
    int64_t total, share;            // tiles in all, tiles of a CTA
    __device__ __forceinline__ Stretch(int tiles, int units, int ctas) {
        total = static_cast<int64_t>(tiles) * units;
        share = max((total + ctas - 1) / ctas, static_cast<int64_t>(1));
    }
};
struct Pair {
    int seq, unit, tiles;            // unit: key head and 16 of its query heads
    int64_t begin;                   // of its tiles in the line
};
__device__ __forceinline__ Pair find_pair(const int* first, int num_seqs, int units, int64_t tile) {
    int lo = 0, hi = num_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (static_cast<int64_t>(first[mid]) * units <= tile) lo = mid;
        else hi = mid;
    }
    // (of sequences without tiles, which start where the next one does, the last is found, which has some)
    const int n = first[lo + 1] - first[lo];
    const int64_t at = static_cast<int64_t>(first[lo]) * units;
    const int unit = static_cast<int>((tile - at) / n);
    return Pair{lo, unit, n, at + static_cast<int64_t>(unit) * n};
}
__device__ __forceinline__ int chunks_of(const PagedAttentionArgs& a) { return (a.heads / a.kv_heads + kHeadRows - 1) / kHeadRows; }

// ------------------------------------------------------------------------------------------------ a stretch of one pair
template <int kDim>
struct WarpState {
    float o[kDim / 8][4], top[2], sum[2];
};
template <int kDim, int kWarps>
__device__ __forceinline__ void attend(const PagedAttentionArgs& a, uint8_t* ring, uint32_t* bad_tiles, int seq, int kv_head, int head0, int rows, int tile0, int tile1,
                                       WarpState<kDim>& st) {
    using Shape = PagedShape<kDim, kWarps>;
    constexpr int kTileKeys = Shape::kTileKeys;
    constexpr int kPieces = kDim / 8, kPassRows = 32 / kPieces;      // 16-byte pieces of a row, rows of one copy instruction
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int keys = keys_of(a, seq), pieces = a.dim / 8;
    uint8_t* mine = ring + warp * Shape::kWarpBytes;
    const uint32_t base = ptx::smem_u32(mine);
    // queries: rows are heads
    uint32_t q[kDim / 16][4];
    {
        const bf16* p = static_cast<const bf16*>(a.q.data) + seq * a.q.stride_token;
#pragma unroll
        for (int k = 0; k < kDim / 16; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = (lane >> 2) + (i & 1) * 8, c = k * 16 + (lane & 3) * 2 + (i >> 1) * 8;
                q[k][i] = row < rows && c < a.dim ? *reinterpret_cast<const uint32_t*>(p + (head0 + row) * a.q.stride_head + c) : 0u;
            }
    }
#pragma unroll
    for (int i = 0; i < kDim / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) st.o[i][j] = 0.f;
    st.top[0] = st.top[1] = kLowest;
    st.sum[0] = st.sum[1] = 0.f;

    const bf16 *k_head = static_cast<const bf16*>(a.k_cache) + kv_head * a.stride_head, *v_head = static_cast<const bf16*>(a.v_cache) + kv_head * a.stride_head;
    const int32_t* table = a.page_table + seq * a.table_pitch;
    // lanes 0 to 15: a key of the tile, and its page, which may be any number
    auto key_of = [&](int tile) { return tile * kTileKeys + warp * 16 + (lane & 15); };
    auto page_of = [&](int tile) { return tile < tile1 && key_of(tile) < keys ? table[static_cast<uint32_t>(key_of(tile)) / static_cast<uint32_t>(a.page_size)] : -1; };
    int page = page_of(tile0);
    auto request = [&](int tile, int stage) {
        if (tile < tile1) {
            const int key = key_of(tile);
            const bool there = page >= 0 && page < a.num_pages;
            const int64_t at = there ? page * a.stride_page + static_cast<int64_t>(static_cast<uint32_t>(key) % static_cast<uint32_t>(a.page_size)) * a.stride_slot : -1;
            // keys of the sequence whose page is none
            const uint32_t bad = __ballot_sync(0xffffffffu, !there && key < keys) & 0xffffu;
            if (lane == 0) bad_tiles[warp * kPagedStages + stage] = bad;
            page = page_of(tile + 1);
            const uint32_t to = base + stage * Shape::kStageBytes;
            const int piece = lane % kPieces;
#pragma unroll
            for (int i = 0; i < 16 / kPassRows; ++i) {
                const int row = i * kPassRows + lane / kPieces;
                const int64_t from = __shfl_sync(0xffffffffu, at, row);
                const uint32_t dst = to + row * Shape::kRowBytes + ((piece ^ (row & 7)) * 16);
                if (piece < pieces) {
                    copy16(dst, k_head + max(from, static_cast<int64_t>(0)) + piece * 8, from >= 0);
                    copy16(dst + 16 * Shape::kRowBytes, v_head + max(from, static_cast<int64_t>(0)) + piece * 8, from >= 0);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // channels that the heads do not have stay zero
    if (pieces < kPieces) {
        for (int i = lane; i < Shape::kWarpBytes / 16; i += 32) *reinterpret_cast<uint4*>(mine + i * 16) = make_uint4(0, 0, 0, 0);
        __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < kPagedStages - 1; ++i) request(tile0 + i, i);
    const float c = a.scale * kPagedLog2e;
    int stage = 0;
    for (int tile = tile0; tile < tile1; ++tile) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kPagedStages - 2) : "memory");
        __syncwarp();
        request(tile + kPagedStages - 1, stage == 0 ? kPagedStages - 1 : stage - 1);
        const uint32_t from = base + stage * Shape::kStageBytes;
        float s[2][4] = {};
        const int r = lane & 7, m = lane >> 3;
#pragma unroll
        for (int k = 0; k < kDim / 16; ++k) {
            uint32_t b[4];
            const int row = (m >> 1) * 8 + r, piece = k * 2 + (m & 1);
            matrices(b, from + row * Shape::kRowBytes + ((piece ^ (row & 7)) * 16));
            mma(s[0], q[k], b[0], b[1]);
            mma(s[1], q[k], b[2], b[3]);
        }
        const int key0 = tile * kTileKeys + warp * 16 + (lane & 3) * 2;
        const uint32_t bad = bad_tiles[warp * kPagedStages + stage];
        if (tile * kTileKeys + warp * 16 + 16 > keys || bad != 0) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = j * 8 + (i & 1);
                    if (key0 + key >= keys) s[j][i] = kLowest;
                    else if (bad >> (key + (lane & 3) * 2) & 1) s[j][i] = __int_as_float(0x7fc00000);
                }
        }
        uint32_t p[4];
        bool move = false;
        float top[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float t = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
            // the reference moves only when the largest score is more than 2^8 above it
            const bool up = (t - st.top[h]) * c > 8.f || st.top[h] == kLowest;
            top[h] = up ? t : st.top[h];
            move |= up && t != kLowest;
        }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float factor = top[h] == st.top[h] ? 1.f : ex2((st.top[h] - top[h]) * c);
                st.sum[h] *= factor;
                st.top[h] = top[h];
#pragma unroll
                for (int i = 0; i < kDim / 8; ++i) {
                    st.o[i][2 * h] *= factor;
                    st.o[i][2 * h + 1] *= factor;
                }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float minus = st.top[h] == kLowest ? 0.f : -st.top[h] * c;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float x = ex2(fmaf(s[j][2 * h], c, minus)), y = ex2(fmaf(s[j][2 * h + 1], c, minus));
                st.sum[h] += x + y;
                p[j * 2 + h] = pack2(x, y);
            }
        }
#pragma unroll
        for (int n = 0; n < kDim / 16; ++n) {
            uint32_t b[4];
            const int row = (m & 1) * 8 + r, piece = n * 2 + (m >> 1);
            matrices_transposed(b, from + 16 * Shape::kRowBytes + row * Shape::kRowBytes + ((piece ^ (row & 7)) * 16));
            mma(st.o[2 * n], p, b[0], b[1]);
            mma(st.o[2 * n + 1], p, b[2], b[3]);
        }
        stage = stage + 1 == kPagedStages ? 0 : stage + 1;
        __syncwarp();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        st.sum[h] += __shfl_xor_sync(0xffffffffu, st.sum[h], 1);
        st.sum[h] += __shfl_xor_sync(0xffffffffu, st.sum[h], 2);
    }
}

// Result (part == null) or part of a pair, from its warps' states
template <int kDim, int kWarps>
__device__ __forceinline__ void join_warps(const PagedAttentionArgs& a, uint8_t* ring, float* s_top, float* s_sum, const WarpState<kDim>& st, int seq, int head0, int rows,
                                           float* part, bool broken) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float c = a.scale * kPagedLog2e;
    __syncthreads();
    if ((lane & 3) == 0)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            s_top[warp * kHeadRows + h * 8 + (lane >> 2)] = st.top[h];
            s_sum[warp * kHeadRows + h * 8 + (lane >> 2)] = broken ? __int_as_float(0x7fc00000) : st.sum[h];
        }
    __syncthreads();
    float* sums = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = h * 8 + (lane >> 2);
        float top = kLowest;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_top[w * kHeadRows + row]);
        const float factor = st.top[h] == kLowest ? 0.f : ex2((st.top[h] - top) * c);
        if (row < rows)
#pragma unroll
            for (int i = 0; i < kDim / 8; ++i)
                *reinterpret_cast<float2*>(sums + (warp * kHeadRows + row) * kDim + i * 8 + (lane & 3) * 2) = make_float2(st.o[i][2 * h] * factor, st.o[i][2 * h + 1] * factor);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * (kDim / 4); i += kWarps * 32) {
        const int row = i / (kDim / 4), d = i % (kDim / 4) * 4;
        float top = kLowest, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_top[w * kHeadRows + row]);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float t = s_top[w * kHeadRows + row], u = s_sum[w * kHeadRows + row];
            sum += t == kLowest && u == 0.f ? 0.f : u * ex2((t - top) * c);
            const float4 x = *reinterpret_cast<const float4*>(sums + (w * kHeadRows + row) * kDim + d);
            v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
        }
        if (part != nullptr) {
            *reinterpret_cast<float4*>(part + row * kDim + d) = v;
            if (d == 0) {
                part[kHeadRows * kDim + row] = top;
                part[kHeadRows * kDim + kHeadRows + row] = sum;
            }
        } else if (d < a.dim) {
            const float inv = 1.f / sum;
            *reinterpret_cast<uint2*>(static_cast<bf16*>(a.o) + (static_cast<int64_t>(seq) * a.heads + head0 + row) * a.dim + d) =
                make_uint2(pack2(v.x * inv, v.y * inv), pack2(v.z * inv, v.w * inv));
        }
    }
    __syncthreads();
}

template <int kThreads>
__device__ __forceinline__ void clear_results(const PagedAttentionArgs& a, int seq) {
    uint2* out = reinterpret_cast<uint2*>(static_cast<bf16*>(a.o) + static_cast<int64_t>(seq) * a.heads * a.dim);
    const uint32_t v = a.lengths[seq] > 0 ? 0x7fc07fc0u : 0u;      // (a table without places)
    for (int i = threadIdx.x; i < a.heads * a.dim / 4; i += kThreads) out[i] = make_uint2(v, v);
}

// kSplit: a CTA takes an equal stretch of all tiles; otherwise it takes a pair
template <int kDim, int kWarps, bool kSplit>
__global__ void __launch_bounds__(kWarps * 32, PagedShape<kDim, kWarps>::kCtas) paged_attention_kernel(const __grid_constant__ PagedAttentionArgs a) {
    using Shape = PagedShape<kDim, kWarps>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_top[kWarps * kHeadRows], s_sum[kWarps * kHeadRows];
    __shared__ uint32_t s_bad[kWarps * kPagedStages];
    const int chunks = chunks_of(a), units = a.kv_heads * chunks, group = a.heads / a.kv_heads;
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    auto run = [&](int seq, int unit, int tile0, int tile1, float* part) {
        const int kv_head = unit / chunks, first = (unit - kv_head * chunks) * kHeadRows, rows = min(group - first, kHeadRows);
        WarpState<kDim> st;
        attend<kDim, kWarps>(a, smem, s_bad, seq, kv_head, kv_head * group + first, rows, tile0, tile1, st);
        join_warps<kDim, kWarps>(a, smem, s_top, s_sum, st, seq, kv_head * group + first, rows, part, a.lengths[seq] > capacity(a));
    };
    if constexpr (kSplit) {
        int4 open = make_int4(0, 0, 0, 0);           // the pair that begins here and ends in a later stretch: sequence, unit, last stretch, whether there is one
        int* first = reinterpret_cast<int*>(smem + Shape::kRing);
        count_tiles<Shape::kThreads, Shape::kTileKeys>(a, first);
        const Stretch all(first[a.num_seqs], units, gridDim.x);
        int64_t at = all.share * blockIdx.x;
        const int64_t end = min(at + all.share, all.total);
        const int64_t begin = at;
        while (at < end) {
            const Pair p = find_pair(first, a.num_seqs, units, at);
            const int64_t until = min(p.begin + p.tiles, end);
            const bool whole = at == p.begin && until == p.begin + p.tiles;
            float* part = whole ? nullptr : a.parts + (static_cast<int64_t>(blockIdx.x) * 2 + (p.begin >= begin ? 1 : 0)) * Shape::kPartFloats;
            run(p.seq, p.unit, static_cast<int>(at - p.begin), static_cast<int>(until - p.begin), part);
            if (!whole && p.begin >= begin) open = make_int4(p.seq, p.unit, static_cast<int>((p.begin + p.tiles - 1) / all.share), 1);
            at = until;
        }
        if (threadIdx.x == 0) a.open_pairs[blockIdx.x] = open;
        for (int seq = blockIdx.x; seq < a.num_seqs; seq += gridDim.x)
            if (first[seq + 1] == first[seq]) clear_results<Shape::kThreads>(a, seq);
    } else {
        const int seq = blockIdx.x / units, tiles = tiles_of_keys<Shape::kTileKeys>(keys_of(a, seq));
        if (tiles > 0) run(seq, blockIdx.x % units, 0, tiles, nullptr);
        else if (blockIdx.x % units == 0) clear_results<Shape::kThreads>(a, seq);
    }
}

// Joins the pair that begins in stretch blockIdx.x and ends in a later one: warps_per_head of eight warps add up the parts of a head
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32;
template <int kDim, int kWarps>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ PagedAttentionArgs a, int warps_per_head) {
    using Shape = PagedShape<kDim, kWarps>;
    constexpr int kPer = kDim / 32;                  // channels of a lane
    __shared__ float s_sum[kJoinWarps], s_value[kJoinWarps][kDim];
    ptx::wait_for_previous_kernel();
    ptx::let_next_kernel_start();
    const int4 p = a.open_pairs[blockIdx.x];
    if (p.w == 0) return;
    const int last = p.z, chunks = chunks_of(a), group = a.heads / a.kv_heads;
    const int kv_head = p.y / chunks, chunk = p.y - kv_head * chunks, rows = min(group - chunk * kHeadRows, kHeadRows);
    const float c = a.scale * kPagedLog2e;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.y * (kJoinWarps / warps_per_head) + warp / warps_per_head, mine = warp % warps_per_head;
    const bool in = row < rows;
    auto part = [&](int cta) { return a.parts + (static_cast<int64_t>(cta) * 2 + (cta == static_cast<int>(blockIdx.x) ? 1 : 0)) * Shape::kPartFloats; };
    float sum = 0.f, v[kPer] = {};
    if (in) {
        float top = kLowest;
#pragma unroll 8
        for (int cta = blockIdx.x + lane; cta <= last; cta += 32) top = fmaxf(top, part(cta)[kHeadRows * kDim + row]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll 8
        for (int cta = blockIdx.x + mine; cta <= last; cta += warps_per_head) {
            const float* from = part(cta);
            const float t = from[kHeadRows * kDim + row], u = from[kHeadRows * kDim + kHeadRows + row];
            const float factor = t == kLowest ? 0.f : ex2((t - top) * c);
            sum += t == kLowest ? u * 0.f : u * factor;      // (a broken part's total is no number)
            float x[kPer];
            if constexpr (kPer == 4) *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(from + row * kDim + lane * 4);
            else *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(from + row * kDim + lane * 2);
#pragma unroll
            for (int i = 0; i < kPer; ++i) v[i] = fmaf(x[i], factor, v[i]);
        }
    }
    if (lane == 0) s_sum[warp] = sum;
#pragma unroll
    for (int i = 0; i < kPer; ++i) s_value[warp][lane * kPer + i] = v[i];
    __syncthreads();
    if (!in || mine != 0) return;
    for (int w = 1; w < warps_per_head; ++w) {
        sum += s_sum[warp + w];
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] += s_value[warp + w][lane * kPer + i];
    }
    const float inv = 1.f / sum;
    if (lane * kPer < a.dim) {
        bf16* out = static_cast<bf16*>(a.o) + (static_cast<int64_t>(p.x) * a.heads + kv_head * group + chunk * kHeadRows + row) * a.dim + lane * kPer;
#pragma unroll
        for (int i = 0; i < kPer; i += 2) *reinterpret_cast<uint32_t*>(out + i) = pack2(v[i] * inv, v[i + 1] * inv);
    }
}

// ------------------------------------------------------------------------------------------------ host
int units_of(const PagedAttentionArgs& a) { return a.kv_heads * ((a.heads / a.kv_heads + kHeadRows - 1) / kHeadRows); }
int64_t capacity_of(const PagedAttentionArgs& a) { return static_cast<int64_t>(a.table_width) * a.page_size; }
// Sequences that cannot be long: a CTA per pair, and nothing to join
bool in_pairs(const PagedAttentionArgs& a) { return capacity_of(a) <= kPairKeys; }
// Where pairs are many, most of what a CTA does is to begin and to end one: CTAs of one warp, eight times as many, do so beside one another.  Few pairs are cut into fewer stretches by
// CTAs of four warps, whose parts are fewer to join.
bool by_warps(const PagedAttentionArgs& a, int num_sms) { return static_cast<int64_t>(a.num_seqs) * units_of(a) >= kManyPairs * num_sms; }
template <class Shape>
int stretches(const PagedAttentionArgs& a, int num_sms) {
    const int64_t most = (capacity_of(a) + Shape::kTileKeys - 1) / Shape::kTileKeys * a.num_seqs * units_of(a);
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(num_sms * Shape::kCtas, most)));
}
template <int kDim, int kWarps>
cudaError_t launch(PagedAttentionArgs a, int num_sms, cudaStream_t stream) {
    using Shape = PagedShape<kDim, kWarps>;
    const bool pairs = in_pairs(a);
    const void* fn = pairs ? reinterpret_cast<const void*>(paged_attention_kernel<kDim, kWarps, false>) : reinterpret_cast<const void*>(paged_attention_kernel<kDim, kWarps, true>);
    const int counts = (a.num_seqs + 1) * 4;
    const int most = Shape::kRing + (EP_MAX_PAGED_SEQS + 1) * 4;
    static std::atomic<uint64_t> allowed[2];
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) return err;
    if (device >= 64 || (allowed[pairs].load(std::memory_order_relaxed) >> device & 1) == 0) {
        err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (err != cudaSuccess) {
            cudaGetLastError();      // the caller reports it
            return err;
        }
        if (device < 64) allowed[pairs].fetch_or(1ull << device, std::memory_order_relaxed);
    }
    void* params[] = {&a};
    const int64_t num_pairs = static_cast<int64_t>(a.num_seqs) * units_of(a);
    if (pairs) return launch_dependent(fn, dim3(static_cast<unsigned>(num_pairs)), dim3(Shape::kThreads), params, Shape::kRing, stream);
    const int ctas = stretches<Shape>(a, num_sms);
    a.open_pairs = reinterpret_cast<int4*>(a.parts + static_cast<int64_t>(ctas) * 2 * Shape::kPartFloats);
    err = launch_dependent(fn, dim3(ctas), dim3(Shape::kThreads), params, Shape::kRing + counts, stream);
    if (err != cudaSuccess) return err;
    // warps for the parts that a pair may have
    int warps_per_head = 1;
    while (warps_per_head < kJoinWarps && ctas / num_pairs >= 8 * warps_per_head) warps_per_head *= 2;
    const int heads = std::min(a.heads / a.kv_heads, kHeadRows), per_cta = kJoinWarps / warps_per_head;
    void* join_params[] = {&a, &warps_per_head};
    return launch_dependent(reinterpret_cast<const void*>(paged_join_kernel<kDim, kWarps>), dim3(ctas, (heads + per_cta - 1) / per_cta), dim3(kJoinThreads), join_params, 0, stream);
}
template <class F>
auto with_shape(const PagedAttentionArgs& a, int num_sms, F f) {
    using One = std::integral_constant<int, 1>;
    using Four = std::integral_constant<int, 4>;
    if (a.dim <= 64) return by_warps(a, num_sms) ? f(std::integral_constant<int, 64>{}, One{}) : f(std::integral_constant<int, 64>{}, Four{});
    return by_warps(a, num_sms) ? f(std::integral_constant<int, 128>{}, One{}) : f(std::integral_constant<int, 128>{}, Four{});
}

}  // namespace

int64_t paged_attention_workspace(const PagedAttentionArgs& a, int num_sms) {
    if (in_pairs(a)) return 0;
    return with_shape(a, num_sms, [&](auto dim, auto warps) {
        using Shape = PagedShape<decltype(dim)::value, decltype(warps)::value>;
        return static_cast<int64_t>(stretches<Shape>(a, num_sms)) * (2 * Shape::kPartFloats * 4 + 16);      // (parts, then open_pairs)
    });
}
cudaError_t launch_paged_attention(const PagedAttentionArgs& a, int num_sms, cudaStream_t stream) {
    return with_shape(a, num_sms, [&](auto dim, auto warps) { return launch<decltype(dim)::value, decltype(warps)::value>(a, num_sms, stream); });
}

}  // namespace ep
