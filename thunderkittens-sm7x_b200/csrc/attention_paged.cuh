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
// Bytes go through shared memory, a ring of kStages x 16 tokens for each warp alone
// (cp.async and __syncwarp, no CTA barrier): what HBM needs in flight, some 100 KB an SM,
// does not fit the registers. The ring's 16-byte pieces are swizzled so that both the
// K reads (rows g, pieces 2t) and the V reads (rows 2t, pieces g) hit distinct banks.
//
// Long contexts are cut into `splits` chunks, each a CTA of its own, whose (max, sum, O)
// a second kernel joins in chunk order: results do not depend on timing.
#pragma once

#include <atomic>

#include "attention.cuh"
#include "kvcache.cuh"

namespace tk {
namespace paged {

using attn::ex2;

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kStep = 16;       // tokens per warp step
constexpr int kCtasPerSm = 24;
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
    int tiles;          // row tiles per (request, key head)
    int splits, chunk;  // chunks per (request, key head, tile), and tokens in each (the last takes the rest)
    float scale, softcap;
    const float* slopes;
    float* part_o;      // [item][rows][D], unnormalised, splits > 1
    float2* part_ml;    // [item][rows]: reference point (log2 units), sum
};

struct Request {
    int first, n, len;  // first query token, how many, tokens in the cache
};

// What the lengths of request r mean, with every index kept inside the arrays.
__device__ __forceinline__ Request request_of(const Params& p, int r) {
    Request q;
    const int a = max(p.starts[r], 0), b = min(p.starts[r + 1], p.n_tokens);
    const long long most = static_cast<long long>(p.width) * p.page;
    q.len = static_cast<int>(min(static_cast<long long>(max(p.seq_lens[r], 0)), most));
    q.first = a;
    q.n = max(b - a, 0);
    return q;
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

// tanh(x) = 1 - 2 / (1 + e^2x), 1 and -1 where the exponential is infinite or 0; absolute
// error about 2^-22.
__device__ __forceinline__ float tanh_of(float x) {
    return fmaf(-2.0f, rcp_approx(1.0f + ex2(x * (2.0f * kLog2e))), 1.0f);
}

// 16 tokens of one key head in a warp's ring: K, then V, 16 D bytes each, in lines of 128
// bytes (a token, or two of head_dim 64). Piece c of token r stands at piece_at.
template <int D, bool kV>
__device__ __forceinline__ uint32_t piece_at(int r, int c) {
    if constexpr (D == 128) return r * 128 + ((c ^ (kV ? r & 6 : r & 1)) << 4);
    return (r >> 1) * 128 + ((((r & 1) * 4 + c) ^ (kV ? r & 6 : 0)) << 4);
}

// What comes with 16 tokens in registers.
struct Step {
    float ks, vs;
    bool on;  // the page is there
};

template <int D>
__device__ __forceinline__ void load_step(Step& st, uint32_t stage, const Params& p, int head, int page, int token, int lane) {
    st.on = page >= 0 && page < p.n_pages;
    if (st.on) {
        const long long tile = static_cast<long long>(page) * p.heads_kv + head;
        const long long at = (tile * p.page + (token & (p.page - 1))) * D + lane * 16;
        constexpr int kPieces = D / 16;             // of a token
        constexpr int kRows = 32 / kPieces;         // tokens per instruction
        const int r = lane / kPieces, c = lane % kPieces;
#pragma unroll
        for (int i = 0; i < kStep / kRows; ++i)
            cp_async_16(stage + piece_at<D, false>(r + i * kRows, c), p.k_cache + at + i * 512);
#pragma unroll
        for (int i = 0; i < kStep / kRows; ++i)
            cp_async_16(stage + kStep * D + piece_at<D, true>(r + i * kRows, c), p.v_cache + at + i * 512);
        st.ks = __ldg(p.k_scale + tile);
        st.vs = __ldg(p.v_scale + tile);
    }
    cp_async_commit();
}

// What one lane knows of its 2 NT score columns (rows 8 nt + 2 t + {0, 1}).
template <int NT>
struct Rows {
    float factor[NT][2];  // of the raw product: softmax scale (log2 units unless scores are changed) and Q's own
    float slope[NT][2];   // log2 units
    int pos[NT][2];       // position, -1 for a row that is not there
    float m[NT][2];       // reference point
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

template <int D>
constexpr int kStages = D == 128 ? 3 : 4;
template <int D, int NT>
constexpr int kSmemBytes = kWarps * kStages<D> * kStep * 2 * D > kWarps * 8 * NT * ((D + 4) * 4 + 8)
                               ? kWarps * kStages<D> * kStep * 2 * D : kWarps * 8 * NT * ((D + 4) * 4 + 8);

template <int D, int NT, bool kBf16, bool kChange>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 4 : 3) paged_kernel(const Params p) {
    constexpr int kRows = 8 * NT;
    constexpr int kM = D / 16;          // MMA tiles of output dims; k-steps of S^T
    constexpr int kPitch = D + 4;       // floats: rows 2t of a store fall on other banks
    extern __shared__ __align__(128) uint8_t smem[];
    // After the loop the rings' memory holds each warp's O, and the (point, sum) of its rows.
    float (*s_o)[kRows][kPitch] = reinterpret_cast<float (*)[kRows][kPitch]>(smem);
    float2 (*s_ml)[kRows] = reinterpret_cast<float2 (*)[kRows]>(smem + kWarps * kRows * kPitch * 4);

    const int lane = static_cast<int>(lane_id());
    const int warp = static_cast<int>(threadIdx.x >> 5);
    const int g = lane >> 2, t = lane & 3;
    int rest = static_cast<int>(blockIdx.x);
    const int split = rest % p.splits;
    rest /= p.splits;
    const int tile = rest % p.tiles;
    rest /= p.tiles;
    const int head = rest % p.heads_kv;
    const int r = rest / p.heads_kv;
    const Request rq = request_of(p, r);
    const int n_rows = min(kRows, rq.n * p.group - tile * kRows);  // of this tile
    if (n_rows <= 0) return;
    // Keys up to the last row's position.
    const int last_pos = rq.len - rq.n + (tile * kRows + n_rows - 1) / p.group;
    const int kv_end = max(last_pos + 1, 0);
    const int begin = split * p.chunk;
    const int end = split == p.splits - 1 ? kv_end : min(kv_end, begin + p.chunk);
    if (begin >= end && split > 0) return;

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
            const uint4 v = there ? __ldg(reinterpret_cast<const uint4*>(at) + i) : make_uint4(0, 0, 0, 0);
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
                                    ? __ldg(p.slopes + head * p.group + row % p.group) * kLog2e : 0.0f;
            rows.m[nt][c] = -INFINITY;
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
    // O is held in units of v_unit, a power of two not below any page scale met so far,
    // so that probabilities times page scale / unit stay in binary16's range.
    float v_unit = 0.0f, v_over = 0.0f;

    const int* table = p.table + static_cast<long long>(r) * p.width;
    auto page_at = [&](int token) { return token < end ? __ldg(table + (token >> p.page_shift)) : -1; };

    auto compute = [&](const Step& st, uint32_t stage, int token) {
        if (!st.on) return;  // no such page: as if its tokens were not there
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[nt][c] = 0.0f;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
            uint32_t near[4], far[4];  // tokens g and g + 8
            load_shared(near, stage + piece_at<D, false>(g, t * (D / 64) + c));
            load_shared(far, stage + piece_at<D, false>(g + 8, t * (D / 64) + c));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int w = 4 * c + i;
                const uint32_t a0 = kv::from_e4m3x2(near[i] & 0xffffu), a2 = kv::from_e4m3x2(near[i] >> 16);
                const uint32_t a1 = kv::from_e4m3x2(far[i] & 0xffffu), a3 = kv::from_e4m3x2(far[i] >> 16);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_16816(s[nt], a0, a1, a2, a3, q[nt][2 * w], q[nt][2 * w + 1]);
            }
        }
        const bool partial = token + kStep > end || token + kStep - 1 > first_pos;
        bool grow = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float x = s[nt][c] * (st.ks * rows.factor[nt][c & 1]);
                const int j = token + g + (c >> 1) * 8;
                if constexpr (kChange) {
                    if (cap > 0.0f) x = cap * tanh_of(x * over_cap);
                    x = fmaf(static_cast<float>(j - rows.pos[nt][c & 1]), rows.slope[nt][c & 1], x * kLog2e);
                }
                if (partial && (j >= end || j > rows.pos[nt][c & 1])) x = -INFINITY;
                s[nt][c] = x;
            }
            grow = grow || fmaxf(s[nt][0], s[nt][2]) > rows.m[nt][0] + 8.0f || fmaxf(s[nt][1], s[nt][3]) > rows.m[nt][1] + 8.0f;
        }
        if (__any_sync(0xffffffffu, grow)) {
            // Move the reference points to the max so far.
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float mx = fmaxf(s[nt][c], s[nt][c + 2]);
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    const float now = fmaxf(rows.m[nt][c], mx);
                    const float alpha = now == -INFINITY ? 1.0f : ex2(rows.m[nt][c] - now);
                    rows.m[nt][c] = now;
                    rows.l[nt][c] *= alpha;
#pragma unroll
                    for (int i = 0; i < kM; ++i) {
                        o[nt][i][c] *= alpha;
                        o[nt][i][c + 2] *= alpha;
                    }
                }
            }
        }
        if (st.vs > v_unit) {
            const uint32_t bits = __float_as_uint(st.vs);
            const float unit = __uint_as_float(((bits + 0x7fffffu) & 0xff800000u));  // the next power of two
            const float alpha = v_unit > 0.0f ? __fdiv_rn(v_unit, unit) : 1.0f;
            v_unit = unit;
            v_over = __fdiv_rn(1.0f, unit);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < kM; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[nt][i][c] *= alpha;
        }
        const float vr = st.vs * v_over;
        uint32_t b[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float e[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float m = rows.m[nt][c & 1];
                e[c] = ex2(s[nt][c] - (m == -INFINITY ? 0.0f : m) + kLift);
            }
            rows.l[nt][0] += e[0] + e[2];
            rows.l[nt][1] += e[1] + e[3];
            b[nt][0] = transpose_8x8(attn::pack_half2(e[0] * vr, e[1] * vr));
            b[nt][1] = transpose_8x8(attn::pack_half2(e[2] * vr, e[3] * vr));
        }
        uint32_t v[4][D / 32];  // tokens 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int r = 2 * t + (u & 1) + (u >> 1) * 8;
            if constexpr (D == 128) load_shared(v[u], stage + kStep * D + piece_at<D, true>(r, g));
            else load_shared(v[u], stage + kStep * D + piece_at<D, true>(r, g >> 1) + (g & 1) * 8);
        }
        if (token + kStep > end) {
            // Places behind the last token hold anything, NaN included: they become 0.
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (token + 2 * t + (u & 1) + (u >> 1) * 8 >= end)
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) v[u][i] = 0;
        }
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            // Bytes 0..3 of a word: dims 4 i .. 4 i + 3 of the lane's D / 8.
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t pick = half == 0 ? 0x5140u : 0x7362u;
                const uint32_t near = __byte_perm(v[0][i], v[1][i], pick), far = __byte_perm(v[2][i], v[3][i], pick);
                const uint32_t a0 = kv::from_e4m3x2(near & 0xffffu), a1 = kv::from_e4m3x2(near >> 16);
                const uint32_t a2 = kv::from_e4m3x2(far & 0xffffu), a3 = kv::from_e4m3x2(far >> 16);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_16816(o[nt][2 * i + half], a0, a1, a2, a3, b[nt][0], b[nt][1]);
            }
        }
    };

    // Warp w takes steps w, w + 4, ... of the chunk; kStages - 1 of them are in flight.
    constexpr int kStride = kWarps * kStep;
    constexpr int kRing = kStages<D>;
    const uint32_t ring = smem_u32(smem) + warp * (kRing * kStep * 2 * D);
    Step steps[kRing];
    int token = begin + warp * kStep;
    int load_token = token;
    int next_page = page_at(load_token);
    auto load_next = [&](Step& st, int stage) {
        const int page = next_page;
        const int at = load_token;
        load_token += kStride;
        next_page = page_at(load_token);
        load_step<D>(st, ring + stage * (kStep * 2 * D), p, head, page, at, lane);
    };
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) load_next(steps[i], i);
    while (token < end) {
#pragma unroll
        for (int i = 0; i < kRing; ++i) {
            if (token < end) {
                cp_async_wait<kRing - 2>();
                __syncwarp();  // every lane's copies of this step have landed, and the step before is read
                load_next(steps[(i + kRing - 1) % kRing], (i + kRing - 1) % kRing);
                compute(steps[i], ring + i * (kStep * 2 * D), token);
                token += kStride;
            }
        }
    }
    cp_async_wait<0>();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
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
    const long long item = item_of(p, r, head, tile, split);
    for (int i = static_cast<int>(threadIdx.x); i < kRows * kQuads; i += kThreads) {
        const int row = i / kQuads, col = (i % kQuads) * 4;
        if (row >= n_rows) break;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_ml[w][row].x);
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float2 ml = s_ml[w][row];
            if (ml.x == -INFINITY) continue;
            const float alpha = ex2(ml.x - m);
            l += ml.y * alpha;
            const float4 v = *reinterpret_cast<const float4*>(&s_o[w][row][col]);
            sum.x += v.x * alpha;
            sum.y += v.y * alpha;
            sum.z += v.z * alpha;
            sum.w += v.w * alpha;
        }
        if (p.splits > 1) {
            *reinterpret_cast<float4*>(p.part_o + (item * kRows + row) * D + col) = sum;
            if (col == 0) p.part_ml[item * kRows + row] = make_float2(m, l);
        } else {
            const float inv = l > 0.0f ? __frcp_rn(l) : 0.0f;  // a row without a key is 0
            const int at = tile * kRows + row;
            uint16_t* dst = p.out + (rq.first + at / p.group) * p.out_stride + (head * p.group + at % p.group) * D + col;
            uint2 w;
            w.x = out_bits<kBf16>(sum.x * inv) | static_cast<uint32_t>(out_bits<kBf16>(sum.y * inv)) << 16;
            w.y = out_bits<kBf16>(sum.z * inv) | static_cast<uint32_t>(out_bits<kBf16>(sum.w * inv)) << 16;
            *reinterpret_cast<uint2*>(dst) = w;
        }
    }
}

// Joins the chunks of one (request, key head, row tile), in chunk order. One CTA each;
// a thread owns 4 dims of a row.
template <int D, int NT, bool kBf16>
__global__ void __launch_bounds__(256) join_kernel(const Params p) {
    constexpr int kRows = 8 * NT;
    constexpr int kQuads = D / 4;
    int rest = static_cast<int>(blockIdx.x);
    const int tile = rest % p.tiles;
    rest /= p.tiles;
    const int head = rest % p.heads_kv;
    const int r = rest / p.heads_kv;
    const Request rq = request_of(p, r);
    const int n_rows = min(kRows, rq.n * p.group - tile * kRows);
    if (n_rows <= 0) return;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int kv_end = max(rq.len - rq.n + (tile * kRows + n_rows - 1) / p.group + 1, 0);
    const int used = max(min((kv_end + p.chunk - 1) / p.chunk, p.splits), 1);
    const long long item = item_of(p, r, head, tile, 0);
    for (int i = static_cast<int>(threadIdx.x); i < n_rows * kQuads; i += 256) {
        const int row = i / kQuads, col = (i % kQuads) * 4;
        float m = -INFINITY;
        for (int s = 0; s < used; ++s) m = fmaxf(m, p.part_ml[(item + s) * kRows + row].x);
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float l = 0.0f;
        for (int s = 0; s < used; ++s) {
            const float2 ml = p.part_ml[(item + s) * kRows + row];
            const float4 v = *reinterpret_cast<const float4*>(p.part_o + ((item + s) * kRows + row) * D + col);
            if (ml.x == -INFINITY) continue;
            const float alpha = ex2(ml.x - m);
            l += ml.y * alpha;
            sum.x += v.x * alpha;
            sum.y += v.y * alpha;
            sum.z += v.z * alpha;
            sum.w += v.w * alpha;
        }
        const float inv = l > 0.0f ? __frcp_rn(l) : 0.0f;
        const int at = tile * kRows + row;
        uint16_t* dst = p.out + (rq.first + at / p.group) * p.out_stride + (head * p.group + at % p.group) * D + col;
        uint2 w;
        w.x = out_bits<kBf16>(sum.x * inv) | static_cast<uint32_t>(out_bits<kBf16>(sum.y * inv)) << 16;
        w.y = out_bits<kBf16>(sum.z * inv) | static_cast<uint32_t>(out_bits<kBf16>(sum.w * inv)) << 16;
        *reinterpret_cast<uint2*>(dst) = w;
    }
}

template <int D, int NT, bool kBf16, bool kChange>
cudaError_t launch_one(const Params& p, unsigned items, int device, cudaStream_t stream) {
    static std::atomic<bool> configured[host::kMaxDevices];
    auto kernel = paged_kernel<D, NT, kBf16, kChange>;
    if (!configured[device].load(std::memory_order_acquire)) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes<D, NT>);
        if (e != cudaSuccess) return e;
        configured[device].store(true, std::memory_order_release);
    }
    kernel<<<items * p.splits, kThreads, kSmemBytes<D, NT>, stream>>>(p);
    return cudaGetLastError();
}

template <int D, int NT, bool kBf16>
cudaError_t launch(const Params& p, bool change, unsigned items, int device, cudaStream_t stream) {
    cudaError_t err = change ? launch_one<D, NT, kBf16, true>(p, items, device, stream)
                             : launch_one<D, NT, kBf16, false>(p, items, device, stream);
    if (err != cudaSuccess || p.splits == 1) return err;
    // Programmatic dependent launch: the join's launch overlaps the last chunks.
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(items);
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, join_kernel<D, NT, kBf16>, p);
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
        !(scale - scale == 0.0f) || !(softcap >= 0.0f) || !(softcap - softcap == 0.0f)) {
        return cudaErrorInvalidValue;
    }
    const long long row = static_cast<long long>(heads_q) * dim;
    auto off = [](const void* x, uintptr_t a) { return (reinterpret_cast<uintptr_t>(x) & (a - 1)) != 0; };
    if (q_stride < row || out_stride < row || q_stride % 8 != 0 || out_stride % 8 != 0 || off(q, 16) || off(out, 16) ||
        off(k_cache, 32) || off(v_cache, 32) ||
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
    p.tiles = static_cast<int>(tiles);
    p.scale = scale;
    p.softcap = softcap;
    p.slopes = slopes;
    // Chunks: enough CTAs for several rounds of the GPU, at least 128 tokens each.
    const long long want = (kCtasPerSm * static_cast<long long>(sm_count) + items - 1) / items;
    const long long most = (max_seq_len + 127LL) / 128;
    long long splits = want < most ? want : most;
    if (splits < 1) splits = 1;
    long long chunk = (max_seq_len + splits - 1) / splits;
    chunk = (chunk + 63) / 64 * 64;
    if (chunk < 64) chunk = 64;
    splits = (max_seq_len + chunk - 1) / chunk;
    p.splits = static_cast<int>(splits < 1 ? 1 : splits);
    p.chunk = static_cast<int>(chunk);
    void* scratch = nullptr;
    if (p.splits > 1) {
        const size_t n = static_cast<size_t>(items) * p.splits * 8 * nt;
        err = host::scratch_alloc(&scratch, n * (static_cast<size_t>(dim) * 4 + 8), device, stream);
        if (err != cudaSuccess) return err;
        p.part_o = static_cast<float*>(scratch);
        p.part_ml = reinterpret_cast<float2*>(p.part_o + n * dim);
    }
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
