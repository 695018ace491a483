// attention_paged.cuh — attention of the newest tokens of each request over a paged
// key/value cache held in e4m3 (layout: kvcache.cuh).
//
//   s_ij = scale * ks[page(j), g] * (q_i . k8_j)          g = h / (heads_q / heads_kv)
//   s_ij = softcap * tanh(s_ij / softcap)                 if softcap > 0
//   s_ij -= slope_h * (pos_i - j)                         if slopes are given
//   o_i  = sum_j softmax_j(s_ij) vs[page(j), g] v8_j      over j <= pos_i
//
// The query tokens of request r are its last ones: token i of n stands at position
// len - n + i.
//
// The cache is read once per tile of 8 or 16 query rows (a row: one query token of one
// of the heads that share a key head), so with few query tokens the kernel is bound by
// HBM: 2 * head_dim bytes a cached token and key head. The products run on
// mma.sync.m16n8k16, not tcgen05: with 8 rows the tensor work is 8192 FLOP for the 256
// bytes of a token, 10 % of what the legacy tensor path does in the time HBM delivers
// them, and the 8-bit operands can go from global memory straight to the registers in
// which the instruction wants them.
//
// A warp takes 16 tokens at a time and computes transposed: S^T = K Q^T (tokens x rows,
// K the A operand), O^T += V^T P^T (dims x rows, V^T the A operand). With the tokens
// as M, 8 rows fill N and nothing is padded. Register layouts (lane = 4 g + t):
//  - K: lane holds dims [D/4 t, D/4 (t + 1)) of tokens g and g + 8: word w of each gives
//    both halves of the A fragment of k-step w, when Q's k order is permuted alike.
//  - V: lane holds dims [D/8 g, D/8 (g + 1)) of tokens 2t, 2t + 1, 2t + 8, 2t + 9; byte
//    pairs of two tokens are one register of V^T. Output dims are permuted alike.
//  - P^T as B operand is the transpose of the S^T accumulator: one movmatrix per 8 x 8.
// Bytes go through shared memory, a ring of kStages x 4 KB for each warp alone
// (cp.async and __syncwarp, no CTA barrier): what HBM needs in flight, some 100 KB an SM,
// does not fit the registers. The ring's 16-byte pieces are swizzled so that both the
// K reads (rows g, pieces 2t) and the V reads (rows 2t, pieces g) hit distinct banks.
//
// Long contexts are cut into `splits` chunks, each a CTA of its own. Up to 8 chunks of one
// (request, key head, row tile) form a cluster that joins their (point, sum, O) through
// distributed shared memory; more of them leave theirs in scratch, and a second kernel
// joins those. Either way in chunk order: results do not depend on timing.
//
// Measured on B200, in a graph: 64 requests of 1 to 8192 tokens, 32 heads on 8 of 128, 96 us = 6.0 TB/s (92 % of the
// measured copy bandwidth; 99 to 104 us as a pass among others on a stream, 85 to 88 %); 3 of 30001 to 65536, capped
// scores, 89 us (91 %). With direct loads to registers instead of the ring 137 us for the first. One request of 2048 tokens 6.8 us: a launch
// and the latencies of lengths, pages, cache and the join. Heads of 64 have twice the tokens, so
// twice the softmax, for the same bytes, and reach 47 % (ragged, 5 drafted tokens, slopes) to 70 %.
#pragma once

#include <atomic>

#include "attention.cuh"
#include "kvcache.cuh"

namespace tk {
namespace paged {

using attn::ex2;

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
// A warp step is kSub blocks of 16 tokens: 4 KB of cache, either way.
template <int D>
constexpr int kSub = 128 / D;
template <int D>
constexpr int kStep = 16 * kSub<D>;
template <int D>
constexpr int kStageBytes = kStep<D> * 2 * D;
// Heads of 64 are bound by instructions, and the loop is unrolled over the stages: 376 requests of 572 to
// 1143 tokens, 4 key heads of 64, 36 us with 2 stages, 39 with 3; 64 of up to 8192, 8 key heads, 63 and 70.
template <int D>
constexpr int kStages = D == 64 ? 2 : 3;
constexpr int kMaxCluster = 8;
constexpr long long kMostTokens = 1LL << 30;  // of a context: positions and steps stay far below 2^31
// CTAs wanted where contexts are ragged, in rounds of 4 for each SM. 64 requests of 1 to 8192 tokens, 8
// key heads of 128: 3 / 4 / 6 / 8 rounds 104 / 98 / 97 / 101 us; 256 of up to 512 tokens: 41 / 41 / 41 / 56.
constexpr int kRounds = 6;
// Most cache bytes a CTA of a joining cluster takes (8 of them an item). One request, 8 key heads: 4096
// x 64 7.6 us in a cluster, 7.7 with the second kernel; 4096 x 128 9.1 and 7.5; 8 requests of 4096 x 128 16.0
// and 21.2; 8192 x 128 13.4 and 8.5.
constexpr long long kClusterBytes = 131072;
constexpr float kLog2e = 1.4426950408889634f;
// Probabilities are held in binary16 as 2^(x - m + kLift), with the reference point m
// at most 8 below the row's max: at most 2^15, so that binary16 keeps 11 bits down to
// 2^-21 of the largest.
constexpr float kLift = 7.0f;

struct Params {
    const uint16_t* q;
    long long q_stride;
    uint16_t* out;
    long long out_stride;
    int n_tokens;
    const uint8_t* k_cache;
    const uint8_t* v_cache;
    const float* k_scale;
    const float* v_scale;
    int n_pages, page, page_shift;
    const int* table;
    int width;
    const int* seq_lens;
    const int* starts;
    int n_requests, heads_q, heads_kv, group;
    int rows;           // most rows of a (request, key head): max_query_len * group
    int tiles;          // row tiles per (request, key head)
    int splits, chunk;  // chunks per (request, key head, tile), and tokens in each (the last takes the rest)
    float scale, softcap;
    const float* slopes;
    bool cluster;       // the chunks of an item are one cluster
    float* part_o;      // [item][rows][D], unnormalised; or null
    float2* part_ml;    // [item][rows]: reference point (log2 units), sum
    int join_runs, join_ctas;
};

struct Request {
    int first, n, len;  // first query token, how many, tokens in the cache
};

// What the lengths of request r mean, with every index kept inside the arrays.
__device__ __forceinline__ Request request_of(const Params& p, int r) {
    Request q;
    const int a = max(p.starts[r], 0), b = min(p.starts[r + 1], p.n_tokens);
    q.len = min(max(p.seq_lens[r], 0), p.width * p.page);
    q.first = a;
    q.n = max(b - a, 0);
    return q;
}

// Rows of a tile; those past max_query_len are left out.
template <int kRows>
__device__ __forceinline__ int rows_of(const Params& p, const Request& rq, int tile) {
    return min(kRows, min(rq.n * p.group, p.rows) - tile * kRows);
}

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// kWords 32-bit words of shared memory, aligned to their size.
template <int kWords>
__device__ __forceinline__ void load_shared(uint32_t (&w)[kWords], uint32_t at) {
    if constexpr (kWords == 4) {
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
    } else {
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
    }
}

// tanh(x) to 2^-21 of itself. Below 5/8 a polynomial x Q(x^2) (fitted to the relative error by least squares on
// Chebyshev nodes, reweighted towards equal ripple: 1.1e-7, 2.1e-7 in FP32): a cap far above the scores
// multiplies what is left of them, so an error relative to 1 would grow with the cap. Above it 1 - 2 / (1 + e^2x),
// 1 and -1 where the exponential is infinite or 0. Both are computed, and one is taken.
__device__ __forceinline__ float tanh_of(float x) {
    const float u = x * x;
    float q = fmaf(1.50511920e-2f, u, -5.18220841e-2f);
    q = fmaf(q, u, 1.33045324e-1f);
    q = fmaf(q, u, -3.33319549e-1f);
    q = fmaf(q, u, 9.99999893e-1f);
    const float far = fmaf(-2.0f, rcp_approx(1.0f + ex2(x * (2.0f * kLog2e))), 1.0f);
    return fabsf(x) < 0.625f ? q * x : far;
}

// 1 / x of a power of two from 2^-126 to 2^126; 2^127 of 0.
__device__ __forceinline__ float inverse_of(float x) { return __uint_as_float((254u << 23) - __float_as_uint(x)); }

// 16 tokens of one key head in a warp's ring: K, then V, 16 D bytes each, in lines of 128
// bytes (a token, or two of head_dim 64). Piece c of token r stands at piece_at.
template <int D, bool kV>
__device__ __forceinline__ uint32_t piece_at(int r, int c) {
    if constexpr (D == 128) return r * 128 + ((c ^ (kV ? r & 6 : r & 1)) << 4);
    return (r >> 1) * 128 + ((((r & 1) * 4 + c) ^ (kV ? r & 6 : 0)) << 4);
}

// What comes with a block of 16 tokens in registers.
struct Block {
    float ks, vs;
    bool on;  // the page is there
};

template <int D>
__device__ __forceinline__ void load_block(Block& bl, uint32_t stage, const Params& p, int head, int page, int token, int lane) {
    bl.on = page >= 0 && page < p.n_pages;
    if (bl.on) {
        const long long tile = static_cast<long long>(page) * p.heads_kv + head;
        const long long at = ((tile << p.page_shift) + (token & (p.page - 1))) * D + lane * 16;
        constexpr int kPieces = D / 16;             // of a token
        constexpr int kRows = 32 / kPieces;         // tokens per instruction
        const int r = lane / kPieces, c = lane % kPieces;
        const uint8_t* k = p.k_cache + at;
        const uint8_t* v = p.v_cache + at;
#pragma unroll
        for (int i = 0; i < 16 / kRows; ++i) cp_async_16(stage + piece_at<D, false>(r + i * kRows, c), k + i * 512);
#pragma unroll
        for (int i = 0; i < 16 / kRows; ++i) cp_async_16(stage + 16 * D + piece_at<D, true>(r + i * kRows, c), v + i * 512);
        bl.ks = p.k_scale[tile];
        bl.vs = p.v_scale[tile];
    }
}

// What one lane knows of its 2 NT score columns (rows 8 nt + 2 t + {0, 1}).
template <int NT>
struct Rows {
    float factor[NT][2];  // of the raw product: softmax scale (log2 units unless scores are changed) and Q's own
    float slope[NT][2];   // log2 units
    int pos[NT][2];       // position, -1 for a row that is not there
    float m[NT][2];       // reference point
    float off[NT][2];     // kLift - m; 0 while there is no point
    float l[NT][2];       // this lane's part of the sum
};

// Item index of the partials.
__device__ __forceinline__ long long item_of(const Params& p, int r, int head, int tile, int split) {
    return ((static_cast<long long>(r) * p.heads_kv + head) * p.tiles + tile) * p.splits + split;
}

template <bool kBf16>
__device__ __forceinline__ uint16_t out_bits(float x) {
    if constexpr (kBf16) {
        const __nv_bfloat16 h = __float2bfloat16_rn(x);
        return *reinterpret_cast<const uint16_t*>(&h);
    } else {
        const __half h = __float2half_rn(x);
        return *reinterpret_cast<const uint16_t*>(&h);
    }
}

// (point, sum, O) of a row, merged one by one in a fixed order. A part without a point has met no key, or
// NaN scores alone, which no max finds: then its sum is NaN, and the row's becomes so.
struct Merged {
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    __device__ __forceinline__ void add(float2 ml, float4 v) {
        if (ml.x == -INFINITY && ml.y == 0.0f) return;
        const float now = fmaxf(m, ml.x);
        const float a = ex2(m - now), b = ex2(ml.x - now);  // 0 for the first: m is -inf
        m = now;
        l = l * a + ml.y * b;
        o.x = o.x * a + v.x * b;
        o.y = o.y * a + v.y * b;
        o.z = o.z * a + v.z * b;
        o.w = o.w * a + v.w * b;
    }
};

template <int D, bool kBf16>
__device__ __forceinline__ void write_out(const Params& p, const Request& rq, int head, int row, int col, const Merged& x) {
    const float inv = x.l == 0.0f ? 0.0f : __frcp_rn(x.l);  // a row without a key is 0
    uint16_t* dst = p.out + (rq.first + row / p.group) * p.out_stride + (head * p.group + row % p.group) * D + col;
    uint2 w;
    w.x = out_bits<kBf16>(x.o.x * inv) | static_cast<uint32_t>(out_bits<kBf16>(x.o.y * inv)) << 16;
    w.y = out_bits<kBf16>(x.o.z * inv) | static_cast<uint32_t>(out_bits<kBf16>(x.o.w * inv)) << 16;
    *reinterpret_cast<uint2*>(dst) = w;
}

// Shared memory: the warps' rings; after the loop, in their place, each warp's O rows (D + 4
// floats apart: rows 2t of a store fall on other banks), its (point, sum), and the CTA's.
template <int D, int NT>
struct Smem {
    static constexpr int kRows = 8 * NT;
    static constexpr int kPitch = D + 4;
    static constexpr int kMl = kWarps * kRows * kPitch * 4;
    static constexpr int kCtaO = kMl + kWarps * kRows * 8;
    static constexpr int kCtaMl = kCtaO + kRows * D * 4;
    static constexpr int kAfter = kCtaMl + kRows * 8;
    static constexpr int kRings = kWarps * kStages<D> * kStageBytes<D>;
    static constexpr int kBytes = kRings > kAfter ? kRings : kAfter;
};

template <int D, int NT, bool kBf16, bool kChange>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 4 : 3) paged_kernel(const Params p) {
    constexpr int kRows = 8 * NT;
    constexpr int kM = D / 16;          // MMA tiles of output dims; k-steps of S^T
    using S = Smem<D, NT>;
    extern __shared__ __align__(128) uint8_t smem[];
    float (*s_o)[kRows][S::kPitch] = reinterpret_cast<float (*)[kRows][S::kPitch]>(smem);
    float2 (*s_ml)[kRows] = reinterpret_cast<float2 (*)[kRows]>(smem + S::kMl);

    const int lane = static_cast<int>(lane_id());
    const int warp = static_cast<int>(threadIdx.x >> 5);
    const int g = lane >> 2, t = lane & 3;
    // x: items; y: chunks, so that first all first chunks start, then all second ones, and so on:
    // those that ragged contexts do not reach come last.
    int rest = static_cast<int>(blockIdx.x);
    const int split = static_cast<int>(blockIdx.y);
    const int tile = rest % p.tiles;
    rest /= p.tiles;
    const int head = rest % p.heads_kv;
    const int r = rest / p.heads_kv;
    // The chain to the first bytes of cache is lengths -> pages -> cache. Which table entries a
    // warp starts with does not depend on the lengths: they are fetched together.
    constexpr int kB = kSub<D>;
    constexpr int kStride = kWarps * kStep<D>;
    const int begin = split * p.chunk;
    const int* table = p.table + static_cast<long long>(r) * p.width;
    int page_of[kStages<D>][kB];
    grid_wait();
#pragma unroll
    for (int i = 0; i < kStages<D>; ++i) {
#pragma unroll
        for (int u = 0; u < kB; ++u) {
            const int col = (begin + (i * kWarps + warp) * kStep<D> + 16 * u) >> p.page_shift;
            page_of[i][u] = col < p.width ? table[col] : -1;
        }
    }
    const Request rq = request_of(p, r);
    const int n_rows = rows_of<kRows>(p, rq, tile);
    if (n_rows <= 0) return;
    // Keys up to the last row's position.
    const int last_pos = rq.len - rq.n + (tile * kRows + n_rows - 1) / p.group;
    const int kv_end = max(last_pos + 1, 0);
    const int end = split == p.splits - 1 ? kv_end : min(kv_end, begin + p.chunk);
    if (begin >= end && split > 0 && !p.cluster) return;

    // Warp w takes steps w, w + 4, ... of the chunk; kStages - 1 of them are in flight.
    const uint32_t ring = smem_u32(smem) + warp * (kStages<D> * kStageBytes<D>);
    Block blocks[kStages<D>][kB];
    int token = begin + warp * kStep<D>;
    int load_token = token;
    int next_page[kB];
    auto page_at = [&](int at) { return at < end ? table[at >> p.page_shift] : -1; };
    auto load_pages = [&](Block (&bl)[kB], const int (&pages)[kB], int stage) {
#pragma unroll
        for (int u = 0; u < kB; ++u) {
            const int at = load_token + 16 * u;
            load_block<D>(bl[u], ring + stage * kStageBytes<D> + u * 32 * D, p, head, at < end ? pages[u] : -1, at, lane);
        }
        cp_async_commit();
        load_token += kStride;
    };
#pragma unroll
    for (int i = 0; i < kStages<D> - 1; ++i) load_pages(blocks[i], page_of[i], i);
#pragma unroll
    for (int u = 0; u < kB; ++u) next_page[u] = page_of[kStages<D> - 1][u];

    // Q as B operand: row g of each 8, dims [D/4 t, D/4 (t + 1)).
    uint32_t q[NT][2 * kM];
    float q_own[NT];  // what the row was divided by
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = tile * kRows + nt * 8 + g;
        const bool there = nt * 8 + g < n_rows;
        const uint16_t* at = p.q + (rq.first + row / p.group) * p.q_stride + (head * p.group + row % p.group) * D + t * (D / 4);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const uint4 v = there ? reinterpret_cast<const uint4*>(at)[i] : make_uint4(0, 0, 0, 0);
            q[nt][4 * i] = v.x;
            q[nt][4 * i + 1] = v.y;
            q[nt][4 * i + 2] = v.z;
            q[nt][4 * i + 3] = v.w;
        }
        q_own[nt] = 1.0f;
        if constexpr (kBf16) {
            // bfloat16 rows are divided by a power of two that brings their largest value
            // to [2^14, 2^15): binary16 then holds exactly every value down to 2^-28 of it.
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < 2 * kM; ++i) {
                const float2 f = kv::bf162_bits_to_float2(q[nt][i]);
                top = fmaxf(top, fmaxf(kv::finite_abs(f.x), kv::finite_abs(f.y)));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -100) - 14;
            const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
            q_own[nt] = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
            for (int i = 0; i < 2 * kM; ++i) {
                const float2 f = kv::bf162_bits_to_float2(q[nt][i]);
                q[nt][i] = attn::pack_half2(f.x * down, f.y * down);
            }
        }
    }

    Rows<NT> rows;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int in_tile = nt * 8 + 2 * t + c;
            const int row = tile * kRows + in_tile;
            const float own = __shfl_sync(0xffffffffu, q_own[nt], 4 * (2 * t + c));
            rows.factor[nt][c] = p.scale * own * (kChange ? 1.0f : kLog2e);
            rows.pos[nt][c] = in_tile < n_rows ? rq.len - rq.n + row / p.group : -1;
            rows.slope[nt][c] = kChange && p.slopes != nullptr && in_tile < n_rows
                                    ? p.slopes[head * p.group + row % p.group] * kLog2e : 0.0f;
            rows.m[nt][c] = -INFINITY;
            rows.off[nt][c] = 0.0f;
            rows.l[nt][c] = 0.0f;
        }
    }
    const int first_pos = rq.len - rq.n + tile * kRows / p.group;  // the tile's smallest position
    const float cap = p.softcap, over_cap = cap > 0.0f ? 1.0f / cap : 0.0f;

    float o[NT][kM][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < kM; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[nt][i][c] = 0.0f;
    // O is held in units of v_unit, a power of two, so that probabilities times page scale / unit stay in
    // binary16's range: not below the page's scale, and at most 2^8 above it, so that they keep their 11 bits
    // down to 2^-13 of the largest weight wherever that lies. Pages more than 2^60 below the largest scale met
    // are left at that (v_floor): O may be that much larger than what it is made of, and stays in FP32's range.
    float v_unit = 0.0f, v_floor = 0.0f;

    auto compute = [&](const Block (&bl)[kB], uint32_t stage, int token) {
        float s[kB][NT][4];
#pragma unroll
        for (int u = 0; u < kB; ++u) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 4; ++c) s[u][nt][c] = 0.0f;
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                uint32_t near[4], far[4];  // tokens g and g + 8
                const uint32_t k = stage + u * 32 * D;
                load_shared(near, k + piece_at<D, false>(g, t * (D / 64) + c));
                load_shared(far, k + piece_at<D, false>(g + 8, t * (D / 64) + c));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int w = 4 * c + i;
                    uint32_t a0, a1, a2, a3;
                    kv::from_e4m3x4(near[i], a0, a2);
                    kv::from_e4m3x4(far[i], a1, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_16816(s[u][nt], a0, a1, a2, a3, q[nt][2 * w], q[nt][2 * w + 1]);
                }
            }
        }
        bool partial = token + kStep<D> > end || token + kStep<D> - 1 > first_pos;
#pragma unroll
        for (int u = 0; u < kB; ++u) partial = partial || !bl[u].on;
        bool grow = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int u = 0; u < kB; ++u) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float x = s[u][nt][c] * (bl[u].ks * rows.factor[nt][c & 1]);
                    const int j = token + 16 * u + g + (c >> 1) * 8;
                    if constexpr (kChange) {
                        if (cap > 0.0f) x = cap * tanh_of(x * over_cap);
                        const float far = static_cast<float>(token + 16 * u + g - rows.pos[nt][c & 1]) + (c >> 1) * 8.0f;
                        x = fmaf(far, rows.slope[nt][c & 1], x * kLog2e);
                    }
                    // Without a page a block's tokens are not there, whatever the ring holds.
                    if (partial && (!bl[u].on || j >= end || j > rows.pos[nt][c & 1])) x = -INFINITY;
                    s[u][nt][c] = x;
                    top[c & 1] = fmaxf(top[c & 1], x);
                }
            }
            grow = grow || top[0] > rows.m[nt][0] + 8.0f || top[1] > rows.m[nt][1] + 8.0f;
        }
        if (__any_sync(0xffffffffu, grow)) {
            // Move the reference points to the max so far.
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float mx = fmaxf(s[0][nt][c], s[0][nt][c + 2]);
#pragma unroll
                    for (int u = 1; u < kB; ++u) mx = fmaxf(mx, fmaxf(s[u][nt][c], s[u][nt][c + 2]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    const float now = fmaxf(rows.m[nt][c], mx);
                    const float alpha = now == -INFINITY ? 1.0f : ex2(rows.m[nt][c] - now);
                    rows.m[nt][c] = now;
                    rows.off[nt][c] = now == -INFINITY ? 0.0f : kLift - now;
                    rows.l[nt][c] *= alpha;
#pragma unroll
                    for (int i = 0; i < kM; ++i) {
                        o[nt][i][c] *= alpha;
                        o[nt][i][c + 2] *= alpha;
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kB; ++u) {
            if (!bl[u].on) continue;
            const float vs = fabsf(bl[u].vs);
            if (vs > v_unit || (vs < v_unit * 0x1p-8f && v_unit > v_floor)) {
                // To the next power of two.
                const float to = __uint_as_float((__float_as_uint(vs) + 0x7fffffu) & 0xff800000u);
                v_floor = fmaxf(v_floor, fmaxf(to * 0x1p-60f, 0x1p-126f));
                const float unit = fminf(fmaxf(to, v_floor), 0x1p126f);
                const float alpha = v_unit * inverse_of(unit);
                v_unit = unit;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < kM; ++i)
#pragma unroll
                        for (int c = 0; c < 4; ++c) o[nt][i][c] *= alpha;
            }
            const float vr = bl[u].vs * inverse_of(v_unit);
            uint32_t b[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float e[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) e[c] = ex2(s[u][nt][c] + rows.off[nt][c & 1]);
                rows.l[nt][0] += e[0] + e[2];
                rows.l[nt][1] += e[1] + e[3];
                b[nt][0] = transpose_8x8(attn::pack_half2(e[0] * vr, e[1] * vr));
                b[nt][1] = transpose_8x8(attn::pack_half2(e[2] * vr, e[3] * vr));
            }
            uint32_t v[4][D / 32];  // tokens 2t, 2t + 1, 2t + 8, 2t + 9
            const uint32_t at = stage + u * 32 * D + 16 * D;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 2 * t + (i & 1) + (i >> 1) * 8;
                if constexpr (D == 128) load_shared(v[i], at + piece_at<D, true>(r, g));
                else load_shared(v[i], at + piece_at<D, true>(r, g >> 1) + (g & 1) * 8);
            }
            if (token + 16 * u + 16 > end) {
                // Places behind the last token hold anything, NaN included: they become 0.
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (token + 16 * u + 2 * t + (i & 1) + (i >> 1) * 8 >= end)
#pragma unroll
                        for (int w = 0; w < D / 32; ++w) v[i][w] = 0;
            }
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                // Bytes 0..3 of a word: dims 4 i .. 4 i + 3 of the lane's D / 8.
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t pick = half == 0 ? 0x5140u : 0x7362u;
                    uint32_t a0, a1, a2, a3;
                    kv::from_e4m3x4(__byte_perm(v[0][i], v[1][i], pick), a0, a1);
                    kv::from_e4m3x4(__byte_perm(v[2][i], v[3][i], pick), a2, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_16816(o[nt][2 * i + half], a0, a1, a2, a3, b[nt][0], b[nt][1]);
                }
            }
        }
    };

    while (token < end) {
#pragma unroll
        for (int i = 0; i < kStages<D>; ++i) {
            if (token < end) {
                cp_async_wait<kStages<D> - 2>();
                __syncwarp();  // every lane's copies of this step have landed, and the step before is read
                constexpr int kAhead = kStages<D> - 1;
                int pages[kB];
#pragma unroll
                for (int u = 0; u < kB; ++u) {
                    pages[u] = next_page[u];
                    next_page[u] = page_at(load_token + kStride + 16 * u);
                }
                load_pages(blocks[(i + kAhead) % kStages<D>], pages, (i + kAhead) % kStages<D>);
                compute(blocks[i], ring + i * kStageBytes<D>, token);
                token += kStride;
            }
        }
    }
    cp_async_wait<0>();
    if (!p.cluster) grid_release();
    __syncthreads();

    // Join the four warps, in warp order.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float l = rows.l[nt][c];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            if (g == 0) s_ml[warp][nt * 8 + 2 * t + c] = make_float2(rows.m[nt][c], l);
#pragma unroll
            for (int i = 0; i < kM; ++i) {
                s_o[warp][nt * 8 + 2 * t + c][g * (D / 8) + 2 * i] = o[nt][i][c] * v_unit;
                s_o[warp][nt * 8 + 2 * t + c][g * (D / 8) + 2 * i + 1] = o[nt][i][c + 2] * v_unit;
            }
        }
    }
    __syncthreads();
    constexpr int kQuads = D / 4;
    const int row0 = tile * kRows;
    for (int i = static_cast<int>(threadIdx.x); i < kRows * kQuads; i += kThreads) {
        const int row = i / kQuads, col = (i % kQuads) * 4;
        if (row >= n_rows) break;
        Merged x;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) x.add(s_ml[w][row], *reinterpret_cast<const float4*>(&s_o[w][row][col]));
        if (p.splits == 1) {
            write_out<D, kBf16>(p, rq, head, row0 + row, col, x);
        } else if (p.cluster) {
            *reinterpret_cast<float4*>(smem + S::kCtaO + (row * D + col) * 4) = x.o;
            if (col == 0) *reinterpret_cast<float2*>(smem + S::kCtaMl + row * 8) = make_float2(x.m, x.l);
        } else {
            const long long item = item_of(p, r, head, tile, split);
            *reinterpret_cast<float4*>(p.part_o + (item * kRows + row) * D + col) = x.o;
            if (col == 0) p.part_ml[item * kRows + row] = make_float2(x.m, x.l);
        }
    }
    if (p.cluster) {
        // CTA `split` of the cluster joins every splits-th 4 dims.
        __syncwarp();
        cluster_sync();
        const uint32_t cta_o = smem_u32(smem + S::kCtaO), cta_ml = smem_u32(smem + S::kCtaMl);
        for (int i = static_cast<int>(threadIdx.x) * p.splits + split; i < n_rows * kQuads; i += kThreads * p.splits) {
            const int row = i / kQuads, col = (i % kQuads) * 4;
            float2 ml[kMaxCluster];
            float4 v[kMaxCluster];
#pragma unroll
            for (int s = 0; s < kMaxCluster; ++s) {
                if (s < p.splits) {
                    ml[s] = ld_shared_cluster_f2(mapa_shared(cta_ml + row * 8, s));
                    v[s] = ld_shared_cluster_f4(mapa_shared(cta_o + (row * D + col) * 4, s));
                }
            }
            Merged x;
#pragma unroll
            for (int s = 0; s < kMaxCluster; ++s)
                if (s < p.splits) x.add(ml[s], v[s]);
            write_out<D, kBf16>(p, rq, head, row0 + row, col, x);
        }
        __syncwarp();
        cluster_sync();  // this CTA's shared memory stays until the others have read it
    }
}

// Joins the rows' chunks from scratch. 256 threads share out (row, run of consecutive
// chunks, 4 dims); the runs of a row are joined in order through shared memory. The host
// chooses `join_runs` runs a row (a power of two, about 4 chunks each), so a CTA holds 256 /
// (D / 4 * join_runs) rows, and `join_ctas` CTAs the rows of an item.
constexpr int kJoinThreads = 256;
template <int D, int NT, bool kBf16>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Params p) {
    constexpr int kRows = 8 * NT;
    constexpr int kQuads = D / 4;
    __shared__ float4 s_o[kJoinThreads];
    __shared__ float2 s_ml[kJoinThreads / kQuads];
    int rest = static_cast<int>(blockIdx.x);
    const int part = rest % p.join_ctas;
    rest /= p.join_ctas;
    const int tile = rest % p.tiles;
    rest /= p.tiles;
    const int head = rest % p.heads_kv;
    const int r = rest / p.heads_kv;
    grid_wait();
    const Request rq = request_of(p, r);
    const int n_rows = rows_of<kRows>(p, rq, tile);
    const int runs = p.join_runs;
    const int slot = static_cast<int>(threadIdx.x) / kQuads, quad = static_cast<int>(threadIdx.x) % kQuads;
    const int run = slot % runs, row = part * (kJoinThreads / kQuads / runs) + slot / runs;
    if (part * (kJoinThreads / kQuads / runs) >= n_rows) return;
    const int kv_end = max(rq.len - rq.n + (tile * kRows + n_rows - 1) / p.group + 1, 0);
    const int used = max(min((kv_end + p.chunk - 1) / p.chunk, p.splits), 1);
    const long long item = item_of(p, r, head, tile, 0);
    const int each = (used + runs - 1) / runs;
    const int last = row < n_rows ? min((run + 1) * each, used) : 0;
    const float2* ml_at = p.part_ml + item * kRows + row;
    const float* o_at = p.part_o + (item * kRows + row) * D + quad * 4;
    Merged x;
    for (int s = run * each; s < last; s += 4) {
        float2 ml[4];
        float4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            ml[u] = make_float2(-INFINITY, 0.0f);
            if (s + u < last) {
                ml[u] = ml_at[static_cast<long long>(s + u) * kRows];
                v[u] = *reinterpret_cast<const float4*>(o_at + static_cast<long long>(s + u) * kRows * D);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) x.add(ml[u], v[u]);
    }
    if (runs > 1) {
        s_o[threadIdx.x] = x.o;
        if (quad == 0) s_ml[slot] = make_float2(x.m, x.l);
        __syncthreads();
        if (run == 0)
            for (int k = 1; k < runs && k * each < used; ++k) x.add(s_ml[slot + k], s_o[threadIdx.x + k * kQuads]);
    }
    if (run == 0 && row < n_rows) write_out<D, kBf16>(p, rq, head, tile * kRows + row, quad * 4, x);
}

template <int D, int NT, bool kBf16, bool kChange>
cudaError_t launch_one(const Params& p, unsigned items, int device, cudaStream_t stream) {
    static std::atomic<bool> configured[host::kMaxDevices];
    auto kernel = paged_kernel<D, NT, kBf16, kChange>;
    if (!configured[device].load(std::memory_order_acquire)) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D, NT>::kBytes);
        if (e != cudaSuccess) return e;
        configured[device].store(true, std::memory_order_release);
    }
    const dim3 grid(items, static_cast<unsigned>(p.splits));
    if (!p.cluster) return host::launch_overlapped(kernel, grid, kThreads, Smem<D, NT>::kBytes, stream, p);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Smem<D, NT>::kBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = static_cast<unsigned>(p.splits);
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int D, int NT, bool kBf16>
cudaError_t launch(const Params& p, bool change, unsigned items, int device, cudaStream_t stream) {
    cudaError_t err = change ? launch_one<D, NT, kBf16, true>(p, items, device, stream)
                             : launch_one<D, NT, kBf16, false>(p, items, device, stream);
    if (err != cudaSuccess || p.part_o == nullptr) return err;
    return host::launch_overlapped(join_kernel<D, NT, kBf16>, dim3(items * p.join_ctas), kJoinThreads, 0, stream, p);
}

inline cudaError_t paged_entry(bool bf16, const void* q, long long q_stride, void* out, long long out_stride, int n_tokens,
                               const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                               int n_pages, int page, const int* table, int width, const int* seq_lens, const int* starts,
                               int n_requests, int heads_q, int heads_kv, int dim, int max_query_len, int max_seq_len,
                               float scale, float softcap, const float* slopes, cudaStream_t stream) {
    if (q == nullptr || out == nullptr || k_cache == nullptr || v_cache == nullptr || k_scale == nullptr || v_scale == nullptr ||
        table == nullptr || seq_lens == nullptr || starts == nullptr || n_tokens < 0 || n_pages <= 0 || width <= 0 ||
        n_requests < 0 || heads_q <= 0 || heads_kv <= 0 || heads_q % heads_kv != 0 || (dim != 64 && dim != 128) ||
        (page != 16 && page != 32 && page != 64 && page != 128) || max_query_len < 0 || max_seq_len < 0 ||
        !host::scores_ok(scale, softcap) || static_cast<long long>(width) * page > kMostTokens) {
        return cudaErrorInvalidValue;
    }
    const long long row = static_cast<long long>(heads_q) * dim;
    if (q_stride < row || out_stride < row || q_stride % 8 != 0 || out_stride % 8 != 0 || host::misaligned(q, 16) || host::misaligned(out, 16) ||
        host::misaligned(k_cache, 32) || host::misaligned(v_cache, 32) || host::misaligned(k_scale, 4) || host::misaligned(v_scale, 4) ||
        host::misaligned(table, 4) || host::misaligned(seq_lens, 4) || host::misaligned(starts, 4) || host::misaligned(slopes, 4) ||
        (n_tokens > 0 && (q_stride > LLONG_MAX / 4 / n_tokens || out_stride > LLONG_MAX / 4 / n_tokens)))
        return cudaErrorInvalidValue;
    const size_t tokens = n_tokens > 0 ? static_cast<size_t>(n_tokens - 1) : 0;
    const size_t some = n_tokens > 0 ? 1 : 0;
    const size_t out_bytes = (tokens * out_stride + some * row) * 2;
    const size_t pages = static_cast<size_t>(n_pages) * heads_kv;
    if (host::ranges_overlap(out, out_bytes, q, (tokens * q_stride + some * row) * 2) ||
        host::ranges_overlap(out, out_bytes, k_cache, pages * page * dim) ||
        host::ranges_overlap(out, out_bytes, v_cache, pages * page * dim) ||
        host::ranges_overlap(out, out_bytes, k_scale, pages * 4) || host::ranges_overlap(out, out_bytes, v_scale, pages * 4) ||
        host::ranges_overlap(out, out_bytes, table, static_cast<size_t>(n_requests) * width * 4) ||
        host::ranges_overlap(out, out_bytes, seq_lens, static_cast<size_t>(n_requests) * 4) ||
        host::ranges_overlap(out, out_bytes, starts, (static_cast<size_t>(n_requests) + 1) * 4) ||
        (slopes != nullptr && host::ranges_overlap(out, out_bytes, slopes, static_cast<size_t>(heads_q) * 4)))
        return cudaErrorInvalidValue;
    if (max_seq_len > width * page) max_seq_len = width * page;  // no context is longer
    const int group = heads_q / heads_kv;
    const long long rows = static_cast<long long>(max_query_len) * group;
    const int nt = rows > 8 ? 2 : 1;
    const long long tiles = (rows + 8 * nt - 1) / (8 * nt);
    const long long items = static_cast<long long>(n_requests) * heads_kv * tiles;
    if (items > (1 << 24)) return cudaErrorInvalidValue;
    int device = 0, sm_count = 0;
    cudaError_t err = host::current_device(&device, &sm_count);
    if (err != cudaSuccess) return err;
    static_cast<void>(cudaGetLastError());
    if (items == 0 || n_tokens == 0) return cudaSuccess;

    Params p{};
    p.q = static_cast<const uint16_t*>(q);
    p.q_stride = q_stride;
    p.out = static_cast<uint16_t*>(out);
    p.out_stride = out_stride;
    p.n_tokens = n_tokens;
    p.k_cache = static_cast<const uint8_t*>(k_cache);
    p.v_cache = static_cast<const uint8_t*>(v_cache);
    p.k_scale = k_scale;
    p.v_scale = v_scale;
    p.n_pages = n_pages;
    p.page = page;
    p.page_shift = page == 16 ? 4 : (page == 32 ? 5 : (page == 64 ? 6 : 7));
    p.table = table;
    p.width = width;
    p.seq_lens = seq_lens;
    p.starts = starts;
    p.n_requests = n_requests;
    p.heads_q = heads_q;
    p.heads_kv = heads_kv;
    p.group = group;
    p.rows = static_cast<int>(rows);
    p.tiles = static_cast<int>(tiles);
    p.scale = scale;
    p.softcap = softcap;
    p.slopes = slopes;
    const long long round = 64 * (128 / dim);  // a step of each warp
    auto cut = [&](long long splits) {
        long long chunk = (max_seq_len + splits - 1) / splits;
        chunk = (chunk + round - 1) / round * round;
        if (chunk < round) chunk = round;
        splits = (max_seq_len + chunk - 1) / chunk;
        p.splits = static_cast<int>(splits < 1 ? 1 : splits);
        p.chunk = static_cast<int>(chunk);
    };
    if (items * kMaxCluster <= 4LL * sm_count && max_seq_len <= kMaxCluster * (kClusterBytes / (2 * dim))) {
        // Short and few, all of it resident at once: one launch.
        cut(kMaxCluster);
        p.cluster = p.splits > 1;
    } else {
        // Enough CTAs for several rounds of the GPU (contexts are ragged, and a cluster would
        // hold its SMs until its longest chunk ends), each of at least 1024 tokens, or 64 KB of
        // cache where one request has to fill the GPU. 512 or 1536 tokens instead of 1024, on heads of 64: 16
        // requests of 17 to 4096 tokens, 16 heads, 25.9 or 25.1 us against 24.9, with 5 drafted tokens 28.1
        // or 31.2 against 28.1; 376 of 572 to 1143, 4 heads, 46 or 36 against 36. Chunks of less than that only where even
        // their CTAs are all resident: 148 requests of 1143 tokens, 4 heads of 64, in one chunk each 17.6
        // us, in two 20; 37 of them 11.0 and 9.2. Few requests pay for it, heads of 128, 8192 tokens, 1 / 2 / 8 requests: one
        // key head 8.4 / 14.3 / 14.4 us, eight key heads 9.3 / 14.5 / 28.1 (their bytes: 2.6 / 5.1 / 20.5).
        const long long least = n_requests == 1 ? 32768 / dim : 1024;
        const long long rounds = n_requests < kRounds ? n_requests : kRounds;
        const long long want = rounds * 4LL * sm_count / items;
        long long most = max_seq_len / least;
        if (most <= 1) most = 2 * items <= 4LL * sm_count && max_seq_len > least ? 2 : 1;
        const long long splits = want < most ? want : most;
        cut(splits < 1 ? 1 : splits);
    }
    void* scratch = nullptr;
    if (p.splits > 1 && !p.cluster) {
        const size_t n = static_cast<size_t>(items) * p.splits * 8 * nt;
        err = host::scratch_alloc(&scratch, n * (static_cast<size_t>(dim) * 4 + 8), device, stream);
        if (err != cudaSuccess) return err;
        p.part_o = static_cast<float*>(scratch);
        p.part_ml = reinterpret_cast<float2*>(p.part_o + n * dim);
    }
    p.join_runs = 1;
    while (p.join_runs * 4 < p.splits && p.join_runs * (dim / 4) < kJoinThreads) p.join_runs *= 2;
    const int join_rows = kJoinThreads / (dim / 4) / p.join_runs;
    p.join_ctas = static_cast<int>(((rows < 8 * nt ? rows : 8 * nt) + join_rows - 1) / join_rows);
    const bool change = softcap > 0.0f || slopes != nullptr;
    const unsigned count = static_cast<unsigned>(items);
    const int kind = (dim == 128 ? 4 : 0) + (nt == 2 ? 2 : 0) + (bf16 ? 1 : 0);
    switch (kind) {
        case 0: err = launch<64, 1, false>(p, change, count, device, stream); break;
        case 1: err = launch<64, 1, true>(p, change, count, device, stream); break;
        case 2: err = launch<64, 2, false>(p, change, count, device, stream); break;
        case 3: err = launch<64, 2, true>(p, change, count, device, stream); break;
        case 4: err = launch<128, 1, false>(p, change, count, device, stream); break;
        case 5: err = launch<128, 1, true>(p, change, count, device, stream); break;
        case 6: err = launch<128, 2, false>(p, change, count, device, stream); break;
        default: err = launch<128, 2, true>(p, change, count, device, stream); break;
    }
    if (scratch != nullptr) cudaFreeAsync(scratch, stream);
    if (err != cudaSuccess) return err;
    return cudaGetLastError();
}

}  // namespace paged
}  // namespace tk
