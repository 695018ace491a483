// attention_masked.cuh — attention forward under masks and score changes, on sm_100a:
//
//   s_ij = scale * q_i . k_j
//   s_ij = softcap * tanh(s_ij / softcap)          if softcap > 0
//   s_ij -= slope_h * |pos_i - j|                  if slopes are given
//   o_i  = sum_j softmax_j(s_ij) v_j  over the keys row i may see; 0 if there are none
//
// pos_i = i + seq_kv - seq_q. Every mask offered here leaves each row ONE interval of
// keys [lo_i, hi_i): causal [0, pos + 1), a prefix [0, max(pos + 1, prefix)), documents
// the run of equal ids that holds the row (cut at pos + 1 if causal). So a block of
// 128 keys is either outside the intervals of all rows of a tile (it is not loaded
// and not multiplied), inside all of them (no mask is computed), or on an edge.
//
// The pipeline is that of attention.cuh: persistent CTAs, two 128-row query tiles each,
// one TMA warp, one MMA-issuing thread, two softmax warpgroups, P written back over S
// in tensor memory; see there for the tensor-memory map, the issue order and its
// hazards. What differs:
//  - each of the two tiles has its own range of key blocks, and the item's loads cover
//    both;
//  - binary16 or bfloat16 in and out, any strides of batch, head and row (4-D tensor maps);
//  - the reference point of a row that has not met an allowed key stays -inf;
//  - P is held as 2^(x - m + 7), so that binary16 keeps its 11 bits down to 2^-21 of
//    the row's largest weight;
//  - head_dim up to 64 leaves room in tensor memory for P beside S: S_{j+1} is multiplied
//    while the softmax of S_j runs (see kApart);
//  - the whole MMA warp runs the issuing loop and an elected lane issues, so that descriptors
//    and addresses are warp-uniform: 5-11 % over one lane in a branch of its own;
//  - with documents, warp 10 zeroes the V rows of padding (negative ids) in shared
//    memory before the PV product reads them: 0 * NaN would be NaN.
// What bounds it: the softmax, as in attention.cuh. A block of 128 keys takes a warp 1024 MUFU
// cycles for its exponentials, two warps share each MUFU, and of the rest (loads from tensor
// memory, max, sums, packing, masks, biases, caps) only part overlaps. Measured on B200, causal,
// burst clocks: 2 x 32 heads on 2 x 8, 4096 x 128, no change of scores 245 us (1,120 TFLOP/s), softcap
// 347 us (MUFU floor 115); 11 documents with slopes, 32 heads, 8192 x 64, 122 us (floor 32: 6 blocks an
// item leave its start and end in sight); 64 heads, a prefix, 1001 rows on 2777 keys, 88 us (256
// items on 148 SMs: two rounds).
#pragma once

#include <cuda_bf16.h>

#include <atomic>
#include <climits>

#include "attention.cuh"

namespace tk {
namespace masked {

using attn::ex2;
using attn::fma2;
using attn::kBlockKV;
using attn::kBlockQ;
using attn::kRegsControl;
using attn::kRegsSoftmax;
using attn::kThreads;
using attn::kTmemCols;

constexpr float kLog2e = 1.4426950408889634f;
// K and V bytes of a group of items (make_item). Causal, 2 x 32 heads, 4096 x 128, 16 / 32 / 64 / 96 / 512
// MB: 290 / 289 / 268 / 274 / 279 us; 8 x 32 heads: 1194 / 1199 / 1150 / 1175 / 1223.
constexpr long long kGroupBytes = 64LL << 20;
constexpr float kLift = 7.0f;  // P <= 2^(8 + kLift) = 2^15 < 65504

// kApart (head_dim up to 64): tile g has S in columns [256g, 256g + 128), O in [+128, +192)
// and P in [+192, +256). The softmax releases S as soon as its row is in registers (s_free),
// so the next S is ready when it has finished with this one, and waits for PV_{j-1} (pv_done)
// only before it writes P and rescales O. Otherwise P overwrites S, PV_j has to complete
// before S_{j+1}, and each tile's chain S -> softmax -> PV -> S is serial. 2 x 32 heads, unmasked,
// 4096 x 64: 412 us with P over S, 326 apart. head_dim 16 and 32 run in 64 columns too, which TMA fills with zeros: their
// exponentials bound them all the same (causal, 2 x 32 heads, 4096, head_dim 64 / 32 / 16: 183 / 181 / 181 us, MUFU 115).
template <int kDPad, bool kBf16>
struct Cfg {
    static constexpr bool kApart = kDPad == 64;
    static constexpr int kTileBytes = kBlockQ * kDPad * 2;  // one Q / K / V tile
    static constexpr int kBoxes = kDPad / 64;                // 64-column TMA boxes per tile
    static constexpr int kSlots = kApart ? 8 : 4;            // K / V ring
    static constexpr int kQBuffers = kApart ? 2 : 1;         // the next item's Q loads early
    static constexpr int kQOffset = 0;                       // Q0, Q1 of each buffer
    static constexpr int kKvOffset = kQBuffers * 2 * kTileBytes;
    static constexpr int kBarOffset = kKvOffset + kSlots * kTileBytes;
    static constexpr int kSmemBytes = kBarOffset + 512 + 1024;
    static constexpr uint32_t kPOffset = kApart ? 192u : 0u; // P's columns in a tile's 256
    static constexpr uint32_t kFormat = kBf16 ? (1u << 7) | (1u << 10) : 0u;  // A and B alike
    static constexpr uint32_t kIdescS = idesc_f16_f32(128, kBlockKV, 0, 0) | kFormat;
    static constexpr uint32_t kIdescO = idesc_f16_f32(128, kDPad, 0, 1) | kFormat;
};

struct Params {
    int seq_q, seq_kv, head_dim;
    int item_tiles;         // query tiles of an item: 2, or 1 where that fills the GPU better
    int per_head;           // items of a (batch, head): ceil(seq_q / (128 item_tiles))
    int tile_stride;        // 128-row tiles of a batch row in `tiles`
    int heads_q, heads_kv, group;
    int num_items;          // batch * heads_q * per_head
    int group_bh;           // (batch, head)s per group of items
    int* next_item;         // zeroed counter, or null: item w -> CTA w % grid
    int causal;
    const int* prefix;      // [batch] or null
    const int2* rows;       // documents: [batch, seq] (lo, hi) of each row; or null
    const int4* tiles;      // documents: [batch, tile_stride] (lo, hi, holds padding, 0) of each 128 rows
    float scale;            // of the raw product
    float scale_log2;       // scale * log2(e)
    float softcap;          // 0: none
    const float* slopes;    // [heads_q] or null
    uint16_t* out;
    long long out_b, out_h, out_s;  // strides in elements
    bool out_vec;           // 16-byte stores
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* map, uint32_t bar, int x, int y, int z, int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}

// tcgen05.mma and commit by one elected lane of a converged warp. With the whole warp in the
// issuing loop its operands are warp-uniform.
__device__ __forceinline__ void mma_ss_elect(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void mma_ts_elect(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void commit_elect(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
        : "memory");
}

// A value that all lanes hold alike, in a form the compiler knows to be warp-uniform.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (kBf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        return attn::pack_half2(lo, hi);
    }
}

// ---- documents --------------------------------------------------------------------

// For every position of a packed row: the run of equal ids that holds it (empty where the id
// is negative), cut at the position itself under a causal mask; then the intervals' hull
// for each 128 rows. One CTA per 1024 positions: a running maximum of run starts, and unless
// causal a running minimum of run ends, inside them; what it needs of the positions outside
// it looks for 4096 at a time. Also zeroes the item counter. 8192 positions: 16 us in one
// CTA, 4.7 us in eight.
constexpr int kRunThreads = 1024;
constexpr int kRunLook = 4;  // positions a thread looks at in a search step

template <bool kMax>
__device__ __forceinline__ int extreme(int a, int b) { return kMax ? max(a, b) : min(a, b); }

// Inclusive running max (kMax, from thread 0 up) or min (from the last thread down) over the CTA;
// `all` is the extreme of every thread's value.
template <bool kMax>
__device__ __forceinline__ int block_running(int v, int* warp_values, int& all) {
    const int lane = static_cast<int>(lane_id());
    const int warp = static_cast<int>(threadIdx.x >> 5);
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int other = kMax ? __shfl_up_sync(0xffffffffu, x, o) : __shfl_down_sync(0xffffffffu, x, o);
        if (kMax ? lane >= o : lane + o < 32) x = extreme<kMax>(x, other);
    }
    if (lane == (kMax ? 31 : 0)) warp_values[warp] = x;
    __syncthreads();
    int y = warp_values[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int other = kMax ? __shfl_up_sync(0xffffffffu, y, o) : __shfl_down_sync(0xffffffffu, y, o);
        if (kMax ? lane >= o : lane + o < 32) y = extreme<kMax>(y, other);
    }
    all = __shfl_sync(0xffffffffu, y, kMax ? 31 : 0);
    const int outer = __shfl_sync(0xffffffffu, y, kMax ? max(warp - 1, 0) : min(warp + 1, 31));
    __syncthreads();
    return warp == (kMax ? 0 : 31) ? x : extreme<kMax>(x, outer);
}

__global__ void __launch_bounds__(kRunThreads) runs_kernel(const int* ids, int seq, int n_tiles, int causal,
                                                           int2* rows, int4* tiles, int* next_item) {
    __shared__ int warp_values[32];
    grid_release();
    grid_wait();
    const int tid = static_cast<int>(threadIdx.x);
    const int s0 = static_cast<int>(blockIdx.x) * kRunThreads;
    const int s = s0 + tid;
    ids += static_cast<long long>(blockIdx.y) * seq;
    rows += static_cast<long long>(blockIdx.y) * seq;
    tiles += static_cast<long long>(blockIdx.y) * n_tiles;
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0 && next_item != nullptr) *next_item = 0;
    const bool there = s < seq;
    const int id = there ? ids[s] : -1;
    const bool starts = there && (s == 0 || ids[s - 1] != id);
    const bool ends = there && (s == seq - 1 || ids[s + 1] != id);
    int all;
    int start = block_running<true>(starts ? s : -1, warp_values, all);
    if (s0 < seq && s0 > 0 && __syncthreads_or(tid == 0 && !starts)) {
        // The first run began before: look back for its start.
        int found = -1;
        for (int hi = s0; found < 0; hi -= kRunThreads * kRunLook) {
            int best = -1;
#pragma unroll
            for (int i = 0; i < kRunLook; ++i) {
                const int k = hi - 1 - (i * kRunThreads + tid);
                if (k >= 0 && (k == 0 || ids[k - 1] != ids[k])) best = max(best, k);
            }
            block_running<true>(best, warp_values, found);
        }
        start = max(start, found);
    }
    int end = s + 1;
    if (causal == 0) {
        end = block_running<false>(ends ? s + 1 : INT_MAX, warp_values, all);
        const int next = min(s0 + kRunThreads, seq);
        if (__syncthreads_or(s == next - 1 && !ends)) {
            // The last run goes on: look for its end.
            int found = INT_MAX;
            for (int lo = next; found == INT_MAX; lo += kRunThreads * kRunLook) {
                int best = INT_MAX;
#pragma unroll
                for (int i = 0; i < kRunLook; ++i) {
                    const int k = lo + i * kRunThreads + tid;
                    if (k < seq && (k == seq - 1 || ids[k + 1] != ids[k])) best = min(best, k + 1);
                }
                block_running<false>(best, warp_values, found);
            }
            end = min(end, found);
        }
    }
    const bool sees = there && id >= 0;
    if (there) rows[s] = sees ? make_int2(start, end) : make_int2(0, 0);
    // Hull of each 128 rows: four warps.
    __shared__ int4 warp_hull[32];
    int lo = sees ? start : INT_MAX, hi = sees ? end : 0, pad = there && id < 0 ? 1 : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        pad |= __shfl_xor_sync(0xffffffffu, pad, o);
    }
    if (lane_id() == 0) warp_hull[tid >> 5] = make_int4(lo, hi, pad, 0);
    __syncthreads();
    const int tile = s0 / kBlockQ + tid;
    if (tid < kRunThreads / kBlockQ && tile < n_tiles) {
        int4 h = warp_hull[4 * tid];
#pragma unroll
        for (int i = 1; i < 4; ++i) {
            const int4 x = warp_hull[4 * tid + i];
            h.x = min(h.x, x.x);
            h.y = max(h.y, x.y);
            h.z |= x.z;
        }
        tiles[tile] = h;
    }
}

__global__ void zero_kernel(int* counter) {
    grid_release();
    grid_wait();
    *counter = 0;
}

// ---- work items ---------------------------------------------------------------------

// One (batch, head) and one or two 128-row query tiles. Items are numbered group by group of
// (batch, head)s, and within a group the last rows of all its heads first: under a
// causal mask those see the most keys, so the GPU runs out of work on the lightest items. A
// group's K and V take half of L2. Tile g works on key blocks [b0[g], b1[g]) (empty if b0 >= b1); the
// item's loads cover [jb, je).
// The TMA thread works an item out and leaves it in shared memory for the other warps.
struct Item {
    int batch, head, q0;
    int tiles;  // of 128 query rows: 1 or 2
    int b0[2], b1[2];
    int jb, je;
    int none;  // no item: the end
};

__device__ __forceinline__ Item make_item(int w, const Params& p) {
    Item it;
    const int first = w / (p.group_bh * p.per_head) * p.group_bh;  // of the group
    const int heads = min(p.group_bh, p.num_items / p.per_head - first);
    const int in_group = w - first * p.per_head;
    const int part = p.per_head - 1 - in_group / heads;
    const int bh = first + in_group % heads;
    it.batch = bh / p.heads_q;
    it.head = bh % p.heads_q;
    it.q0 = part * p.item_tiles * kBlockQ;
    it.tiles = it.q0 + kBlockQ < p.seq_q ? p.item_tiles : 1;
    it.jb = INT_MAX;
    it.je = 0;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const int r0 = it.q0 + g * kBlockQ;
        int lo = 0, hi = 0;
        if (g < it.tiles) {
            if (p.tiles != nullptr) {
                const int4 t = p.tiles[static_cast<long long>(it.batch) * p.tile_stride + part * p.item_tiles + g];
                lo = t.x;
                hi = t.y;
            } else {
                hi = p.seq_kv;
                if (p.causal) {
                    hi = min(r0 + kBlockQ, p.seq_q) + (p.seq_kv - p.seq_q);
                    if (p.prefix != nullptr) hi = max(hi, p.prefix[it.batch]);
                    hi = min(max(hi, 0), p.seq_kv);
                }
            }
        }
        it.b0[g] = lo < hi ? lo / kBlockKV : 0;
        it.b1[g] = lo < hi ? (hi + kBlockKV - 1) / kBlockKV : 0;
        if (it.b0[g] < it.b1[g]) {
            it.jb = min(it.jb, it.b0[g]);
            it.je = max(it.je, it.b1[g]);
        }
    }
    if (it.je == 0) it.jb = 0;
    it.none = 0;
    return it;
}

// ---- scores ---------------------------------------------------------------------------

// A block's 128 keys in four chunks of 32, for the rows of a warp: which chunks hold a masked
// key (`edge`), and which some row sees at all (`live`). [lo, hi) is relative to the block.
struct Chunks {
    uint32_t edge, live;
};

__device__ __forceinline__ Chunks chunks_of(int lo, int hi) {
    Chunks k{0, 0};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (__any_sync(0xffffffffu, lo > 32 * c || hi < 32 * c + 32)) k.edge |= 1u << c;
        if (__any_sync(0xffffffffu, lo < 32 * c + 32 && hi > 32 * c && lo < hi)) k.live |= 1u << c;
    }
    return k;
}

// Keys outside [lo, hi) become -inf, in the chunks that hold some.
__device__ __forceinline__ void mask_row(uint32_t (&r)[128], const Chunks& k, int lo, int hi) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (!(k.edge >> c & 1)) continue;
#pragma unroll
        for (int i = 32 * c; i < 32 * c + 32; ++i)
            if (i < lo || i >= hi) r[i] = 0xff800000u;
    }
}

// 2^(s c + a) of the row's 128 scores; writes them, rounded to 16 bits, to the 64 columns at
// p_addr, and returns their sum. kSkip: chunks of 32 that no row of the warp sees are 0 at once,
// for a branch at each chunk. Where blocks are mostly seen whole the branches cost more (unmasked
// head_dim 64: 363 against 325 us); with documents they pay (138 against 148 us), and so do they
// for capped scores, whose whole blocks go another way. Both forms in one kernel lose to
// either alone there (391 against 355 us): each is 64 pairs of code.
template <bool kBf16, bool kSkip, class Mid>
__device__ __forceinline__ float exp_store(uint32_t p_addr, const uint32_t (&r)[128], float c, float a, uint32_t live, Mid&& mid) {
    float2 acc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t] = make_float2(0.0f, 0.0f);
    const float2 c2 = make_float2(c, c), a2 = make_float2(a, a);
#pragma unroll
    for (int chunk = 0; chunk < 4; ++chunk) {
        if (chunk == 2) mid();
        uint32_t pk[16];
        if (kSkip && !(live >> chunk & 1)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) pk[i] = 0;
            tmem_st_32x32b_x16(p_addr + 16 * chunk, pk);
            continue;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int idx = 32 * chunk + 2 * i;
            const float2 x = fma2(make_float2(__uint_as_float(r[idx]), __uint_as_float(r[idx + 1])), c2, a2);
            const float2 e = make_float2(ex2(x.x), ex2(x.y));
            acc[i & 3] = attn::add2(acc[i & 3], e);
            pk[i] = pack2<kBf16>(e.x, e.y);
        }
        tmem_st_32x32b_x16(p_addr + 16 * chunk, pk);
    }
    const float2 t = attn::add2(attn::add2(acc[0], acc[1]), attn::add2(acc[2], acc[3]));
    return t.x + t.y;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t d;
    asm("{\n\t.reg .b64 ra, rb;\n\tmov.b64 ra, {%1, %2};\n\tmov.b64 rb, {%3, %4};\n\t"
        "mul.rn.f32x2 %0, ra, rb;\n\t}"
        : "=l"(d)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(d));
    return r;
}

// ---- softcap * tanh(s scale / softcap), in log2 units
//
// With z = 8/3 y, y = s scale / softcap:
//   kNear: where all scores of a warp have |y| < 3/4, tanh(y) = z Q(z^2) on the FMA pipe, Q a
//     polynomial of 5 coefficients (a least-squares fit of the relative error on Chebyshev nodes,
//     reweighted towards equal ripple; 5.7e-7, 7.3e-7 in FP32). The limit is |z| < 2, one bit of the
//     exponent, so testing a row is an OR over it.
//   kFar: elsewhere 1 - 2 / (1 + e^2y), four scores to one reciprocal (of the product of their
//     denominators): 1.25 MUFU operations a score beside the softmax's own. e^2y is cut at 2^30, where
//     tanh is 1 in FP32, so that the product stays below 2^121.
// The range is a warp's, for its 128 keys: taken for each 32 keys it was slower wherever one range held
// throughout (384 and 495 us for the next two figures). 2 x 32 heads on 2 x 8, causal, 4096 x 128: no cap 246 us; cap 50,
// standard deviation of the scores 6, near: 348; cap 10, far: 465 (617 with a reciprocal a score in a pass
// of its own; 450 with a second polynomial where |y| < 8/5 suffices, which leaves 617 beyond it); cap 30,
// both ranges along a row: 560, since the two loops share an instruction cache that holds one.
//   kBoth: each value as its own size asks, for caps above kFineCap: kFar is off by softcap * 2^-22 however small
//     the score, and a row of small scores may share a warp with one of large scores.
enum CapRange { kNear, kFar, kBoth };
constexpr float kFineCap = 256.0f;  // kFar is off by 2^-14 at most up to here

// r *= k; whether all of the warp's |r| are below 2 then.
__device__ __forceinline__ bool scale_row(uint32_t (&r)[128], float k) {
    const float2 k2 = make_float2(k, k);
    uint32_t any[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 64; ++i) {
        const float2 z = mul2(make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), k2);
        r[2 * i] = __float_as_uint(z.x);
        r[2 * i + 1] = __float_as_uint(z.y);
        any[i & 3] |= r[2 * i] | r[2 * i + 1];
    }
    return !__any_sync(0xffffffffu, ((any[0] | any[1]) | (any[2] | any[3])) & 0x40000000u);
}

// Scores to z, and the range the warp's lie in. kSteps: scale, then cap, where their quotient is below what
// FP32 holds.
template <bool kSteps>
__device__ __forceinline__ CapRange cap_range(uint32_t (&r)[128], float scale, float softcap) {
    if (kSteps && fabsf(scale) < softcap * 0x1p-125f) {
#pragma unroll
        for (int i = 0; i < 128; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * scale);
        scale = 1.0f;
    }
    return scale_row(r, 8.0f / 3.0f * (scale / softcap)) ? kNear : kFar;
}

constexpr float kCapArg = 0.75f * kLog2e;  // e^2y = 2^(kCapArg z)

// The capped score of one value; out = softcap * log2(e).
__device__ __forceinline__ float cap_one(float z, float out) {
    return fmaf(-2.0f * out, rcp_approx(1.0f + ex2(z * kCapArg)), out);
}

// Capped scores plus a of four values at a time.
template <CapRange kRange>
struct Cap4;

template <>
struct Cap4<kNear> {
    float2 co[5], a2;
    __device__ __forceinline__ Cap4(float out, float a) : a2(make_float2(a, a)) {
        constexpr float near[5] = {3.74999791e-1f, -1.75754447e-2f, 9.83255915e-4f, -5.22008486e-5f, 1.89612661e-6f};
#pragma unroll
        for (int n = 0; n < 5; ++n) co[n] = make_float2(near[n] * out, near[n] * out);
    }
    __device__ __forceinline__ void operator()(float2& z0, float2& z1) const {
        z0 = one(z0);
        z1 = one(z1);
    }
    __device__ __forceinline__ float2 one(float2 z) const {
        const float2 u = mul2(z, z);
        float2 q = fma2(co[4], u, co[3]);
#pragma unroll
        for (int n = 2; n >= 0; --n) q = fma2(q, u, co[n]);
        return fma2(q, z, a2);
    }
};

template <>
struct Cap4<kFar> {
    float2 twice, a2;
    __device__ __forceinline__ Cap4(float out, float a) : twice(make_float2(-2.0f * out, -2.0f * out)), a2(make_float2(out + a, out + a)) {}
    static __device__ __forceinline__ float cut(float t) {  // NaN stays NaN
        float r;
        asm("min.NaN.f32 %0, %1, 0f41F00000;" : "=f"(r) : "f"(t));
        return r;
    }
    __device__ __forceinline__ float2 denominators(float2 z) const {
        const float2 t = mul2(z, make_float2(kCapArg, kCapArg));
        return attn::add2(make_float2(ex2(cut(t.x)), ex2(cut(t.y))), make_float2(1.0f, 1.0f));
    }
    __device__ __forceinline__ void operator()(float2& z0, float2& z1) const {
        const float2 d0 = denominators(z0), d1 = denominators(z1);
        const float2 d = mul2(d0, d1);
        const float r = rcp_approx(d.x * d.y);
        const float2 pairs = make_float2(r * d.y, r * d.x);  // 1 / (d0 d1)
        z0 = fma2(mul2(pairs, d1), twice, a2);
        z1 = fma2(mul2(pairs, d0), twice, a2);
    }
};

// z to capped scores, in place. kFar and kBoth take a reciprocal a score: a NaN that a mask will hide
// must not reach others.
template <CapRange kRange>
__device__ __forceinline__ void cap_row(uint32_t (&r)[128], float out) {
    const Cap4<kNear> near(out, 0.0f);
    const float2 twice = make_float2(-2.0f * out, -2.0f * out), out2 = make_float2(out, out);
#pragma unroll
    for (int i = 0; i < 128; i += 2) {
        const float2 z = make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1]));
        float2 x;
        if constexpr (kRange == kNear) {
            x = near.one(z);
        } else {
            const float2 t = mul2(z, make_float2(kCapArg, kCapArg));
            const float2 d = attn::add2(make_float2(ex2(t.x), ex2(t.y)), make_float2(1.0f, 1.0f));
            x = fma2(make_float2(rcp_approx(d.x), rcp_approx(d.y)), twice, out2);
            if constexpr (kRange == kBoth) {
                const float2 small = near.one(z);
                if (fabsf(z.x) < 2.0f) x.x = small.x;
                if (fabsf(z.y) < 2.0f) x.y = small.y;
            }
        }
        r[i] = __float_as_uint(x.x);
        r[i + 1] = __float_as_uint(x.y);
    }
}

// exp_store of capped scores straight from z. kNear: -inf becomes a weight of 0.
template <bool kBf16, CapRange kRange, class Mid>
__device__ __forceinline__ float cap_exp_store(uint32_t p_addr, const uint32_t (&r)[128], float out, float a, Mid&& mid) {
    const Cap4<kRange> cap(out, a);
    float2 acc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t] = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int chunk = 0; chunk < 4; ++chunk) {
        if (chunk == 2) mid();
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const int idx = 32 * chunk + 2 * i;
            float2 z0 = make_float2(__uint_as_float(r[idx]), __uint_as_float(r[idx + 1]));
            float2 z1 = make_float2(__uint_as_float(r[idx + 2]), __uint_as_float(r[idx + 3]));
            cap(z0, z1);
            const float2 e0 = make_float2(ex2(z0.x), ex2(z0.y)), e1 = make_float2(ex2(z1.x), ex2(z1.y));
            acc[i & 3] = attn::add2(acc[i & 3], e0);
            acc[(i + 1) & 3] = attn::add2(acc[(i + 1) & 3], e1);
            pk[i] = pack2<kBf16>(e0.x, e0.y);
            pk[i + 1] = pack2<kBf16>(e1.x, e1.y);
        }
        tmem_st_32x32b_x16(p_addr + 16 * chunk, pk);
    }
    const float2 t = attn::add2(attn::add2(acc[0], acc[1]), attn::add2(acc[2], acc[3]));
    return t.x + t.y;
}

// Scores r c - slope |pos - j| in log2 units, in place: leaves r with r c + base that score.
// Where the block lies on one side of the rows of a warp, |pos - j| is linear in j: one
// multiply-add a score by a constant of its column (slope / c), the row's part goes to base.
// `from` = pos - first key of the block.
__device__ __forceinline__ void bias_row(uint32_t (&r)[128], float& c, float& base, float slope, int from, bool left, bool right) {
    const float f = static_cast<float>(from);
    if ((left || right) && c > 1e-12f) {  // else also where the scale is not positive: the max of r c is not that of r
        const float up = left ? slope : -slope;  // per key
        const float up_c = __fdiv_rn(up, c);
#pragma unroll
        for (int i = 0; i < 128; ++i) r[i] = __float_as_uint(fmaf(up_c, static_cast<float>(i), __uint_as_float(r[i])));
        base = -up * f;
        return;
    }
#pragma unroll
    for (int i = 0; i < 128; ++i)
        r[i] = __float_as_uint(fmaf(fabsf(f - static_cast<float>(i)), -slope, __uint_as_float(r[i]) * c));
    c = 1.0f;
}

// ---- kernel ---------------------------------------------------------------------------

// What is done to the scores: kernels of their own, since each pass over a row is unrolled to
// 128 scores and the instruction cache feels it.
enum Kind {
    kPlain,        // a positive scale, folded into the exponent
    kCap,
    kBias,         // slopes, or a non-positive scale
    kCapBias,
    kCapFine,      // a cap above kFineCap, with slopes or without
};

template <int kDPad, bool kBf16, Kind kKind, bool kDocs>
__global__ void __launch_bounds__(kThreads, 1)
    masked_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const Params p) {
    using C = Cfg<kDPad, kBf16>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_base = smem_u32(smem_raw);
    const uint32_t base = (raw_base + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw_base);
    const uint32_t bars = base + C::kBarOffset;
    // Where P overwrites S, its first 64 keys are announced while the others' exponentials run (on
    // s_free, which is not used otherwise), and PV begins on them: 6 % at head_dim 128 (unmasked
    // bfloat16, 2 x 32 heads, 4096: 474 to 443 us). With capped scores it loses 2 %.
    constexpr bool kEarly = !C::kApart && (kKind == kPlain || kKind == kBias);
    constexpr int kSlots = C::kSlots;
    auto kv_full = [&](int s) { return bars + 8u * s; };
    auto kv_empty = [&](int s) { return bars + 8u * (kSlots + s); };
    auto v_clean = [&](int s) { return bars + 8u * (2 * kSlots + s); };  // documents: V slot s has no padding rows left
    constexpr int kB = 3 * kSlots;
    auto q_full = [&](int b) { return bars + 8u * (kB + 16 + b); };
    auto q_empty = [&](int b) { return bars + 8u * (kB + 18 + b); };
    constexpr int kQ = C::kQBuffers;
    auto s_full = [&](int g) { return bars + 8u * (kB + 2 + g); };
    auto p_ready = [&](int g) { return bars + 8u * (kB + 4 + g); };
    auto o_final = [&](int g) { return bars + 8u * (kB + 6 + g); };  // kApart: pv_done, after every PV
    auto o_empty = [&](int g) { return bars + 8u * (kB + 8 + g); };
    auto item_full = [&](int s) { return bars + 8u * (kB + 10 + s); };
    auto item_empty = [&](int s) { return bars + 8u * (kB + 12 + s); };
    auto s_free = [&](int g) { return bars + 8u * (kB + 14 + g); };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kBarOffset + 8 * (kB + 20));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    Item* item_ring = reinterpret_cast<Item*>(tmem_slot + 2);  // two entries
    static_assert(8 * (kB + 20) + 8 + 2 * sizeof(Item) <= 512, "barrier block");

    const uint32_t warp = warp_id();
    const uint32_t lane = lane_id();

    if (threadIdx.x == 0) {
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(kv_full(s), 1);
            mbar_init(kv_empty(s), 1);
            mbar_init(v_clean(s), 1);
        }
        for (int g = 0; g < 2; ++g) {
            mbar_init(q_full(g), 1);
            mbar_init(q_empty(g), 1);
            mbar_init(s_full(g), 1);
            mbar_init(p_ready(g), 4);
            mbar_init(s_free(g), 4);
            mbar_init(o_final(g), 1);
            mbar_init(o_empty(g), 4);
            mbar_init(item_full(g), 1);
            mbar_init(item_empty(g), kDocs ? 10 : 9);  // the MMA thread, eight softmax warps, warp 10
        }
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 9) {
        tmem_alloc<1>(smem_u32(tmem_slot), kTmemCols);
        tmem_relinquish<1>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = static_cast<uint32_t>(uniform(static_cast<int>(*tmem_slot)));
    // The kernel before zeroes the counter and finds the documents.
    grid_wait();

    if (warp >= 8) {
        setmaxnreg_dec<kRegsControl>();
        if (warp == 8) {
            // ---------------- TMA producer and scheduler (one thread) ----------------
            if (lane == 0) {
                tma_prefetch_desc(&map_q);
                tma_prefetch_desc(&map_k);
                tma_prefetch_desc(&map_v);
                int slot = 0;
                uint32_t phase = 0;
                int issued = 0;
                int items = 0;    // published
                int loaded = 0;   // of them with keys, so with Q loaded
                bool ok = true;
                int w = static_cast<int>(blockIdx.x);
                for (int it_slot = 0;; it_slot ^= 1) {
                    if (items > 0) {
                        w = p.next_item != nullptr ? static_cast<int>(gridDim.x) + atomicAdd(p.next_item, 1)
                                                   : w + static_cast<int>(gridDim.x);
                    }
                    Item it;
                    if (w < p.num_items) it = make_item(w, p);
                    else it.none = 1;
                    // Entry it_slot was last used two items ago.
                    if (items >= 2 &&
                        !mbar_wait(item_empty(it_slot), static_cast<uint32_t>((items - 2) >> 1) & 1u,
                                   kFaultProducerWait, abort_flag)) {
                        ok = false;
                        break;
                    }
                    item_ring[it_slot] = it;
                    mbar_arrive(item_full(it_slot));
                    if (it.none) break;
                    ++items;
                    if (it.jb >= it.je) continue;
                    // A Q buffer is free once all S products of the item that had it have completed.
                    const int qb = loaded % kQ;
                    if (loaded >= kQ &&
                        !mbar_wait(q_empty(qb), static_cast<uint32_t>(loaded / kQ - 1) & 1u, kFaultProducerWait, abort_flag)) {
                        ok = false;
                        break;
                    }
                    mbar_arrive_expect_tx(q_full(qb), it.tiles * C::kTileBytes);
                    for (int g = 0; g < it.tiles; ++g)
                        for (int x = 0; x < C::kBoxes; ++x)
                            tma_load_4d(base + C::kQOffset + (2 * qb + g) * C::kTileBytes + x * 16384, &map_q, q_full(qb), x * 64,
                                        it.q0 + g * kBlockQ, it.head, it.batch);
                    ++loaded;
                    for (int j = it.jb; j < it.je && ok; ++j) {
                        for (int which = 0; which < 2; ++which) {  // K then V
                            if (!mbar_wait(kv_empty(slot), phase ^ 1u, kFaultProducerWait, abort_flag)) {
                                ok = false;
                                break;
                            }
                            const uint32_t dst = base + C::kKvOffset + slot * C::kTileBytes;
                            mbar_arrive_expect_tx(kv_full(slot), C::kTileBytes);
                            for (int x = 0; x < C::kBoxes; ++x)
                                tma_load_4d(dst + x * 16384, which == 0 ? &map_k : &map_v, kv_full(slot), x * 64,
                                            j * kBlockKV, it.head / p.group, it.batch);
                            ++issued;
                            if (++slot == kSlots) {
                                slot = 0;
                                phase ^= 1u;
                            }
                        }
                    }
                    if (!ok) break;
                }
                if (!ok) {
                    // Let every issued load land before the CTA may exit: the last Q loads
                    // and the last (up to kSlots) K/V loads.
                    for (int i = loaded > kQ ? loaded - kQ : 0; i < loaded; ++i)
                        mbar_wait(q_full(i % kQ), static_cast<uint32_t>(i / kQ) & 1u, kFaultDrainWait, nullptr);
                    int s = slot;
                    uint32_t ph = phase;
                    for (int i = 0; i < min(issued, kSlots); ++i) {
                        if (--s < 0) {
                            s = kSlots - 1;
                            ph ^= 1u;
                        }
                        mbar_wait(kv_full(s), ph, kFaultDrainWait, nullptr);
                    }
                }
            }
            __syncwarp();
        } else if (warp == 9) {
            // ---------------- MMA issuer (whole warp, an elected lane issues) ----------------
            {
                auto kv_addr = [&](int slot) { return base + C::kKvOffset + slot * C::kTileBytes; };
                // A step inside a tile is a plain add to its descriptor's low bits (16-byte units).
                const uint64_t dq0 = sw128_desc(base + C::kQOffset, 16, 1024);
                uint64_t dq = dq0;  // of the item's buffer
                auto issue_s = [&](int g, uint32_t k_addr) {
                    const uint64_t dk = sw128_desc(k_addr, 16, 1024);
#pragma unroll
                    for (int kk = 0; kk < kDPad / 16; ++kk) {
                        const uint64_t off = static_cast<uint64_t>(((kk >> 2) * 16384 + (kk & 3) * 32) >> 4);
                        mma_ss_elect(tmem + 256u * g, dq + static_cast<uint64_t>(g * (C::kTileBytes >> 4)) + off, dk + off, C::kIdescS, kk > 0 ? 1u : 0u);
                    }
                    commit_elect(s_full(g));
                };
                auto issue_pv = [&](int g, uint32_t v_addr, bool first, int k0, int k1) {
                    const uint64_t dv = sw128_desc(v_addr, 16384, 1024);
#pragma unroll
                    for (int kk = k0; kk < k1; ++kk)
                        mma_ts_elect(tmem + 256u * g + 128u, tmem + 256u * g + C::kPOffset + kk * 8,
                                   dv + static_cast<uint64_t>((kk * 2048) >> 4), C::kIdescO, (!first || kk > 0) ? 1u : 0u);
                };
                uint32_t pr_phase[2] = {0, 0};
                int done[2] = {0, 0};  // items in which tile g has produced an output
                int n_s[2] = {0, 0};   // kApart: S products of tile g
                int kv_base = 0;       // K/V loads of the previous items
                int loaded = 0;
                bool ok = true;
                auto o_free = [&](int g) {
                    return done[g] == 0 ||
                           mbar_wait_warp(o_empty(g), static_cast<uint32_t>(done[g] - 1) & 1u, kFaultAttnWait, abort_flag);
                };
                for (int items = 0, it_slot = 0; ok; it_slot ^= 1, ++items) {
                    if (!mbar_wait_warp(item_full(it_slot), static_cast<uint32_t>(items >> 1) & 1u, kFaultAttnWait, abort_flag))
                        break;
                    Item it = item_ring[it_slot];
                    it.jb = uniform(it.jb);
                    it.je = uniform(it.je);
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        it.b0[g] = uniform(it.b0[g]);
                        it.b1[g] = uniform(it.b1[g]);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(item_empty(it_slot));
                    if (uniform(it.none)) break;
                    if (it.jb >= it.je) continue;
                    auto slot_of = [&](int load) { return (kv_base + load) % kSlots; };
                    auto phase_of = [&](int load) { return static_cast<uint32_t>((kv_base + load) / kSlots) & 1u; };
                    auto act = [&](int g, int j) { return j >= it.b0[g] && j < it.b1[g]; };
                    auto wait_k = [&](int j) {
                        return mbar_wait_warp(kv_full(slot_of(2 * (j - it.jb))), phase_of(2 * (j - it.jb)), kFaultAttnWait, abort_flag);
                    };
                    auto wait_v = [&](int j) {
                        const int load = 2 * (j - it.jb) + 1;
                        return mbar_wait_warp(kDocs ? v_clean(slot_of(load)) : kv_full(slot_of(load)), phase_of(load),
                                         kFaultAttnWait, abort_flag);
                    };
                    // PV of tile g, block j, once its probabilities are there.
                    auto pv = [&](int g, int j) {
                        const bool first = j == it.b0[g];
                        const uint32_t v = kv_addr(slot_of(2 * (j - it.jb) + 1));
                        if constexpr (kEarly) {
                            if (!mbar_wait_warp(s_free(g), pr_phase[g], kFaultAttnWait, abort_flag)) return false;
                            if (first && !o_free(g)) return false;
                            tc_fence_after();
                            issue_pv(g, v, first, 0, 4);
                        }
                        if (!mbar_wait_warp(p_ready(g), pr_phase[g], kFaultAttnWait, abort_flag)) return false;
                        pr_phase[g] ^= 1u;
                        if (!kEarly && first && !o_free(g)) return false;
                        tc_fence_after();
                        if constexpr (kEarly) issue_pv(g, v, false, 4, 8);
                        else issue_pv(g, v, first, 0, 8);
                        if (C::kApart || j == it.b1[g] - 1) commit_elect(o_final(g));
                        return true;
                    };
                    const int qb = loaded % kQ;
                    ok = mbar_wait_warp(q_full(qb), static_cast<uint32_t>(loaded / kQ) & 1u, kFaultAttnWait, abort_flag);
                    dq = dq0 + static_cast<uint64_t>(qb * (2 * C::kTileBytes >> 4));
                    ++loaded;
                    if constexpr (C::kApart) {
                        // Per step: S0_{j+1}, PV1_{j-1}, S1_{j+1}, PV0_j, each as soon as what it
                        // needs is there; the tiles stay half a period apart.
                        auto s_mma = [&](int g, int j) {
                            if (n_s[g] > 0 &&
                                !mbar_wait_warp(s_free(g), static_cast<uint32_t>(n_s[g] - 1) & 1u, kFaultAttnWait, abort_flag))
                                return false;
                            ++n_s[g];
                            tc_fence_after();
                            issue_s(g, kv_addr(slot_of(2 * (j - it.jb))));
                            return true;
                        };
                        for (int j = it.jb - 1; j <= it.je && ok; ++j) {
                            ok = false;
                            const bool more = j + 1 < it.je;
                            if (more && !wait_k(j + 1)) break;
                            if (act(0, j + 1) && !s_mma(0, j + 1)) break;
                            if (j > it.jb) {
                                if (act(1, j - 1) && !pv(1, j - 1)) break;
                                commit_elect(kv_empty(slot_of(2 * (j - 1 - it.jb) + 1)));
                            }
                            if (act(1, j + 1) && !s_mma(1, j + 1)) break;
                            if (more) {
                                commit_elect(kv_empty(slot_of(2 * (j + 1 - it.jb))));
                                if (j + 1 == it.je - 1) commit_elect(q_empty(qb));
                            }
                            if (j >= it.jb && j < it.je) {
                                if (!wait_v(j)) break;
                                if (act(0, j) && !pv(0, j)) break;
                            }
                            ok = true;
                        }
                    } else {
                        if (ok && act(0, it.jb)) {
                            ok = wait_k(it.jb);
                            tc_fence_after();
                            if (ok) issue_s(0, kv_addr(slot_of(0)));
                        }
                        for (int j = it.jb; j < it.je && ok; ++j) {
                            ok = false;
                            const int load = 2 * (j - it.jb);
                            // PV1 of the block before, then its V is free.
                            if (j > it.jb) {
                                if (act(1, j - 1) && !pv(1, j - 1)) break;
                                commit_elect(kv_empty(slot_of(load - 1)));
                            }
                            // S1, then K is free. K was waited for before S0, where tile 0 works on it.
                            if (!act(0, j) && !wait_k(j)) break;
                            if (act(1, j)) {
                                tc_fence_after();
                                issue_s(1, kv_addr(slot_of(load)));
                            }
                            commit_elect(kv_empty(slot_of(load)));
                            if (j == it.je - 1) commit_elect(q_empty(qb));
                            // PV0 and the next block's S0, back to back.
                            if (!wait_v(j)) break;
                            const bool next = act(0, j + 1);
                            if (next && !wait_k(j + 1)) break;
                            if (act(0, j) && !pv(0, j)) break;
                            if (next) {
                                tc_fence_after();
                                issue_s(0, kv_addr(slot_of(load + 2)));
                            }
                            if (j == it.je - 1) {
                                if (act(1, j) && !pv(1, j)) break;
                                commit_elect(kv_empty(slot_of(load + 1)));
                            }
                            ok = true;
                        }
                    }
#pragma unroll
                    for (int g = 0; g < 2; ++g)
                        if (it.b0[g] < it.b1[g]) ++done[g];
                    kv_base += 2 * (it.je - it.jb);
                }
            }
            __syncwarp();
        } else if (kDocs && warp == 10) {
            // ---------------- padding rows of V become 0 ----------------
            int kv_base = 0;
            bool ok = true;
            for (int items = 0, it_slot = 0; ok; it_slot ^= 1, ++items) {
                if (!mbar_wait_warp(item_full(it_slot), static_cast<uint32_t>(items >> 1) & 1u, kFaultAttnWait, abort_flag))
                    break;
                const Item it = item_ring[it_slot];
                __syncwarp();
                if (lane == 0) mbar_arrive(item_empty(it_slot));
                if (it.none) break;
                for (int j = it.jb; j < it.je; ++j) {
                    const int load = kv_base + 2 * (j - it.jb) + 1;
                    const int slot = load % kSlots;
                    if (!mbar_wait_warp(kv_full(slot), static_cast<uint32_t>(load / kSlots) & 1u, kFaultAttnWait, abort_flag)) {
                        ok = false;
                        break;
                    }
                    // Documents have seq_kv = seq_q: key block j holds the rows of tile j.
                    if (p.tiles[static_cast<long long>(it.batch) * p.tile_stride + j].z != 0) {
                        const uint32_t tile = base + C::kKvOffset + slot * C::kTileBytes;
#pragma unroll
                        for (int i = 0; i < kBlockKV / 32; ++i) {
                            const int row = i * 32 + static_cast<int>(lane);
                            const int key = j * kBlockKV + row;
                            if (key >= p.seq_kv) continue;  // zero already
                            const int2 r = p.rows[static_cast<long long>(it.batch) * p.seq_kv + key];
                            if (r.x < r.y) continue;
                            for (int x = 0; x < C::kBoxes; ++x)
#pragma unroll
                                for (int c = 0; c < 8; ++c) st_shared_v4(tile + x * 16384 + row * 128 + c * 16, 0, 0, 0, 0);
                        }
                        fence_proxy_async_smem();
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(v_clean(slot));
                }
                kv_base += 2 * (it.je - it.jb);
            }
        }
    } else {
        setmaxnreg_inc<kRegsSoftmax>();
        // ---------------- softmax warpgroups (warps 0-3: tile 0, 4-7: tile 1) ----------------
        const int g = static_cast<int>(warp >> 2);
        const uint32_t quarter = warp & 3u;
        const int row_in_tile = static_cast<int>(quarter * 32 + lane);
        const uint32_t lane_bits = (quarter * 32u) << 16;
        const uint32_t s_addr = tmem + lane_bits + 256u * g;
        const uint32_t o_addr = s_addr + 128u;
        uint32_t sf_phase = 0;  // s_full(g) completions seen
        uint32_t of_phase = 0;  // o_final(g) completions seen
        bool ok = true;
        for (int it_slot = 0, items = 0; ok; it_slot ^= 1, ++items) {
            if (!mbar_wait_warp(item_full(it_slot), static_cast<uint32_t>(items >> 1) & 1u, kFaultAttnWait, abort_flag))
                break;
            const int none = item_ring[it_slot].none, batch = item_ring[it_slot].batch, head = item_ring[it_slot].head;
            const int q0 = item_ring[it_slot].q0 + g * kBlockQ, tiles = item_ring[it_slot].tiles;
            const int b0 = uniform(item_ring[it_slot].b0[g]), b1 = uniform(item_ring[it_slot].b1[g]);
            __syncwarp();
            if (lane == 0) mbar_arrive(item_empty(it_slot));
            if (uniform(none)) break;
            const int q_row = q0 + row_in_tile;
            if (g >= uniform(tiles)) continue;
            const int pos = q_row + p.seq_kv - p.seq_q;
            // The row's keys [lo, hi). Rows past the end take every key, so that they never
            // make their warp compute a mask; they are not stored.
            int lo = 0, hi = INT_MAX;
            if (q_row < p.seq_q) {
                lo = 0;
                hi = p.seq_kv;
                if constexpr (kDocs) {
                    const int2 r = p.rows[static_cast<long long>(batch) * p.seq_q + q_row];
                    lo = r.x;
                    hi = r.y;
                } else if (p.causal) {
                    hi = pos + 1;
                    if (p.prefix != nullptr) hi = min(max(hi, p.prefix[batch]), p.seq_kv);
                }
            }
            float slope = 0.0f;
            if ((kKind == kBias || kKind == kCapBias || kKind == kCapFine) && p.slopes != nullptr) slope = p.slopes[head] * kLog2e;
            float m_run = -INFINITY;  // reference point, log2 units
            float l_run = 0.0f;       // running sum of 2^(x - m_run + kLift)
            for (int j = b0; j < b1; ++j) {
                if (!mbar_wait_warp(s_full(g), sf_phase, kFaultAttnWait, abort_flag)) {
                    ok = false;
                    break;
                }
                sf_phase ^= 1u;
                tc_fence_after();
                const int kv0 = j * kBlockKV;
                const bool need_mask = __any_sync(0xffffffffu, lo > kv0 || hi < kv0 + kBlockKV);
                uint32_t r[128];
                attn::load_row128(s_addr, r);
                if constexpr (C::kApart) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s_free(g));
                }
                // Scores in log2 units are r * c + base.
                float c = p.scale_log2, base = 0.0f;
                const float cap_out = p.softcap * kLog2e;
                // The chunks are worked out before the bias (122 against 128 us with documents and slopes,
                // 8192 x 64), but after a cap (348 against 352 us).
                constexpr bool kCapped = kKind == kCap || kKind == kCapBias || kKind == kCapFine;
                Chunks chunks{0, 15};
                if (!kCapped && need_mask) chunks = chunks_of(lo - kv0, hi - kv0);
                // Capped scores without a bias go from z to P in one pass, where a masked z of -inf ends as a
                // weight of 0 (kNear) or none is masked. Capping keeps the order, so the row's max is found on z.
                CapRange range = kFar;
                bool fused = false;
                if constexpr (kCapped) {
                    range = cap_range<kKind == kCapFine>(r, p.scale, p.softcap);
                    fused = kKind == kCap && (range == kNear || !need_mask);
                    if (kKind != kCap && range == kNear) {
                        cap_row<kNear>(r, cap_out);
                    } else if (kKind == kCapFine) {
                        cap_row<kBoth>(r, cap_out);
                    } else if (!fused) {
                        cap_row<kFar>(r, cap_out);
                    }
                    c = 1.0f;
                }
                if (kKind == kBias || kKind == kCapBias || (kKind == kCapFine && p.slopes != nullptr)) {
                    // Keys behind the row's position are masked, unless all of them are seen.
                    const bool left = (p.causal && p.prefix == nullptr) || __all_sync(0xffffffffu, kv0 + kBlockKV - 1 <= pos);
                    const bool right = __all_sync(0xffffffffu, kv0 >= pos);
                    bias_row(r, c, base, slope, pos - kv0, left, right);
                }
                if (need_mask) {
                    if (kCapped) chunks = chunks_of(lo - kv0, hi - kv0);
                    mask_row(r, chunks, lo - kv0, hi - kv0);
                }
                const float r_max = attn::row_max128(r);
                const float m_blk = kKind == kCap && fused ? cap_one(r_max, cap_out) : fmaf(r_max, c, base);
                // The point moves only when the max grows by more than 8, so P <= 2^(8 + kLift).
                const float m_new = fmaxf(m_run, m_blk);
                const float m_use = m_new > m_run + 8.0f ? m_new : m_run;
                const float alpha = m_use == m_run ? 1.0f : ex2(m_run - m_use);
                if (C::kApart && j > b0) {
                    // PV_{j-1} has read P and written O.
                    if (!mbar_wait_warp(o_final(g), of_phase, kFaultAttnWait, abort_flag)) {
                        ok = false;
                        break;
                    }
                    of_phase ^= 1u;
                    tc_fence_after();
                }
                // tcgen05.ld/st are warp-collective: the rescale runs for the whole warp when any of
                // its rows needs it. PV_{j-1} has completed (in-order tcgen05, or waited for).
                auto rescale = [&]() {
                    if (j > b0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll
                        for (int x = 0; x < kDPad / 16; ++x) {
                            uint32_t o[16];
                            tmem_ld_32x32b_x16(o_addr + 16 * x, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tmem_st_32x32b_x16(o_addr + 16 * x, o);
                        }
                    }
                };
                if constexpr (kEarly) rescale();
                auto mid = [&]() {
                    if constexpr (kEarly) {
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(s_free(g));
                    }
                };
                const float a = kLift - (m_use == -INFINITY ? 0.0f : m_use);
                float e_sum;
                if (kKind == kCap && fused) {
                    e_sum = range == kNear ? cap_exp_store<kBf16, kNear>(s_addr + C::kPOffset, r, cap_out, a, mid)
                                           : cap_exp_store<kBf16, kFar>(s_addr + C::kPOffset, r, cap_out, a, mid);
                } else {
                    constexpr bool kSkip = kDocs || kCapped;
                    e_sum = exp_store<kBf16, kSkip>(s_addr + C::kPOffset, r, c, base + a, chunks.live, mid);
                }
                if constexpr (!kEarly) rescale();
                l_run = l_run * alpha + e_sum;
                m_run = m_use;
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready(g));
            }
            if (!ok) break;
            const bool row_ok = q_row < p.seq_q;
            uint16_t* orow = p.out + batch * p.out_b + head * p.out_h + static_cast<long long>(q_row) * p.out_s;
            if (b0 >= b1) {
                // No row of the tile sees a key: nothing was multiplied.
                if (row_ok) {
                    for (int col = 0; col < p.head_dim; ++col) orow[col] = 0;
                }
                continue;
            }
            if (!mbar_wait_warp(o_final(g), of_phase, kFaultAttnWait, abort_flag)) {
                ok = false;
                break;
            }
            of_phase ^= 1u;
            tc_fence_after();
            const float inv_l = l_run > 0.0f ? __frcp_rn(l_run) : 0.0f;  // a row without a key is 0
#pragma unroll
            for (int x = 0; x < kDPad / 32; ++x) {
                uint32_t r[32];
                tmem_ld_32x32b_x32(o_addr + 32 * x, r);
                tmem_wait_ld();
                if (x == kDPad / 32 - 1) {
                    // O_g is in registers: the next item's first PV may overwrite it.
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(o_empty(g));
                }
                if (row_ok) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int col = 32 * x + 8 * q;
                        if (col < p.head_dim) {
                            uint32_t w[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                w[i] = pack2<kBf16>(__uint_as_float(r[8 * q + 2 * i]) * inv_l,
                                                    __uint_as_float(r[8 * q + 2 * i + 1]) * inv_l);
                            if (p.out_vec) {
                                *reinterpret_cast<uint4*>(orow + col) = make_uint4(w[0], w[1], w[2], w[3]);
                            } else {
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    orow[col + 2 * i] = static_cast<uint16_t>(w[i]);
                                    orow[col + 2 * i + 1] = static_cast<uint16_t>(w[i] >> 16);
                                }
                            }
                        }
                    }
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc<1>(tmem, kTmemCols);
    }
}

// ---- host -------------------------------------------------------------------------------

// A [batch, heads, rows, dim] operand and its strides in elements (dim: 1).
struct View {
    const void* p;
    long long b, h, s;
};

// Rows TMA cannot address, as a contiguous [batch, heads, rows, dim] copy.
__global__ void gather_rows_kernel(const uint16_t* src, long long sb, long long sh, long long ss, uint16_t* dst, int heads,
                                   int rows, int dim, long long count) {
    for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < count;
         i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int d = static_cast<int>(i % dim);
        const long long row = i / dim;
        const int s = static_cast<int>(row % rows);
        const long long bh = row / rows;
        dst[i] = src[(bh / heads) * sb + (bh % heads) * sh + s * ss + d];
    }
}

template <int kDPad, bool kBf16, Kind kKind, bool kDocs>
cudaError_t launch_kernel(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const Params& p, int device,
                        int grid, cudaStream_t stream) {
    using C = Cfg<kDPad, kBf16>;
    static std::atomic<bool> configured[host::kMaxDevices];
    auto kernel = masked_kernel<kDPad, kBf16, kKind, kDocs>;
    if (!configured[device].load(std::memory_order_acquire)) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
        if (e != cudaSuccess) return e;
        configured[device].store(true, std::memory_order_release);
    }
    return host::launch_overlapped(kernel, dim3(static_cast<unsigned>(grid)), kThreads, C::kSmemBytes, stream, mq, mk, mv, p);
}

template <int kDPad, bool kBf16, Kind kKind>
cudaError_t launch_kind(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const Params& p, int device,
                        int grid, cudaStream_t stream) {
    return p.rows != nullptr ? launch_kernel<kDPad, kBf16, kKind, true>(mq, mk, mv, p, device, grid, stream)
                             : launch_kernel<kDPad, kBf16, kKind, false>(mq, mk, mv, p, device, grid, stream);
}

template <int kDPad, bool kBf16>
cudaError_t launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const Params& p, int device,
                   int grid, cudaStream_t stream) {
    const bool bias = p.slopes != nullptr || (p.softcap == 0.0f && !(p.scale > 0.0f));
    // kCap takes a row's reference point from cap_one and large scores from kFar, both off by softcap * 2^-22 and
    // more; kCapFine takes the point from the capped scores, and those from kBoth. With kBoth in kCapBias, that
    // lost 2 to 8 % for ordinary caps (causal, 2 x 32 heads, 4096 x 128, cap 50, 10: 441, 605 us against 451, 636).
    if (p.softcap > kFineCap) return launch_kind<kDPad, kBf16, kCapFine>(mq, mk, mv, p, device, grid, stream);
    if (p.softcap > 0.0f)
        return bias ? launch_kind<kDPad, kBf16, kCapBias>(mq, mk, mv, p, device, grid, stream)
                    : launch_kind<kDPad, kBf16, kCap>(mq, mk, mv, p, device, grid, stream);
    return bias ? launch_kind<kDPad, kBf16, kBias>(mq, mk, mv, p, device, grid, stream)
                : launch_kind<kDPad, kBf16, kPlain>(mq, mk, mv, p, device, grid, stream);
}

// Strides of a dimension of size 1 are never used; the others have to be positive.
inline bool strides_ok(const View& v, int batch, int heads, int rows) {
    return (batch == 1 || v.b > 0) && (heads == 1 || v.h > 0) && (rows == 1 || v.s > 0);
}

// Elements from the first to behind the last one (saturating far above any allocation).
inline bool extent_of(const View& v, int batch, int heads, int rows, int dim, size_t* elems) {
    const __int128 e = static_cast<__int128>(batch - 1) * (batch > 1 ? v.b : 0) +
                       static_cast<__int128>(heads - 1) * (heads > 1 ? v.h : 0) +
                       static_cast<__int128>(rows - 1) * (rows > 1 ? v.s : 0) + dim;
    if (e > (static_cast<__int128>(1) << 60)) return false;
    *elems = static_cast<size_t>(e);
    return true;
}

// No two (batch, head, row) of an output share an element: taken from the smallest
// stride up, each dimension steps over all that the smaller ones reach.
inline bool rows_apart(const View& v, int batch, int heads, int rows, int dim) {
    long long st[3] = {v.b, v.h, v.s};
    int n[3] = {batch, heads, rows};
    for (int i = 0; i < 2; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (st[j] < st[i]) {
                const long long a = st[i];
                st[i] = st[j];
                st[j] = a;
                const int c = n[i];
                n[i] = n[j];
                n[j] = c;
            }
    __int128 reach = dim;
    for (int i = 0; i < 3; ++i) {
        if (n[i] == 1) continue;
        if (st[i] < reach) return false;
        reach += static_cast<__int128>(n[i] - 1) * st[i];
    }
    return true;
}

inline bool make_map(CUtensorMap* map, const View& v, int batch, int heads, int rows, int dim) {
    const uint64_t dims[4] = {static_cast<uint64_t>(dim), static_cast<uint64_t>(rows), static_cast<uint64_t>(heads),
                              static_cast<uint64_t>(batch)};
    // A dimension of size 1 gets any stride that the encoding takes.
    const uint64_t strides[3] = {rows > 1 ? static_cast<uint64_t>(v.s) * 2 : 256, heads > 1 ? static_cast<uint64_t>(v.h) * 2 : 256,
                                 batch > 1 ? static_cast<uint64_t>(v.b) * 2 : 256};
    const uint32_t box[4] = {64, 128, 1, 1};
    return host::make_map_f16(map, v.p, 4, dims, strides, box);
}

inline cudaError_t masked_entry(bool bf16, const void* q, const void* k, const void* v, void* out, const int64_t* strides,
                                int batch, int heads, int heads_kv, int seq_q, int seq_kv, int dim, float scale, float softcap,
                                const float* slopes, const int* doc_ids, const int* prefix, int causal, cudaStream_t stream) {
    if (q == nullptr || k == nullptr || v == nullptr || out == nullptr || batch <= 0 || heads <= 0 || heads_kv <= 0 ||
        heads % heads_kv != 0 || seq_q <= 0 || seq_kv <= 0 || (dim != 16 && dim != 32 && dim != 64 && dim != 128) ||
        (causal != 0 && causal != 1) || !host::scores_ok(scale, softcap) ||
        (doc_ids != nullptr && (prefix != nullptr || seq_q != seq_kv || batch > 65535)) || (prefix != nullptr && causal == 0)) {
        return cudaErrorInvalidValue;
    }
    if (host::misaligned(q, 2) || host::misaligned(k, 2) || host::misaligned(v, 2) || host::misaligned(out, 2) || host::misaligned(slopes, 4) ||
        host::misaligned(doc_ids, 4) || host::misaligned(prefix, 4)) {
        return cudaErrorInvalidValue;
    }
    // A normal scale / softcap; above kFineCap the kernel divides the scores instead.
    const float size = scale < 0.0f ? -scale : scale;
    if (softcap > 0.0f && softcap <= kFineCap && scale != 0.0f && size < softcap * 0x1p-125f) return cudaErrorInvalidValue;
    const long long bh = static_cast<long long>(batch) * heads;
    const int pairs = static_cast<int>((seq_q + 255LL) / 256);
    // Positions and the last tile's ends stay below 2^31.
    if (bh * pairs > INT_MAX / 2 || seq_q > INT_MAX - 512 || seq_kv > INT_MAX - 512) return cudaErrorInvalidValue;
    const long long dq = static_cast<long long>(seq_q) * dim, dk = static_cast<long long>(seq_kv) * dim;
    View vq{q, heads * dq, dq, dim}, vk{k, heads_kv * dk, dk, dim}, vv{v, heads_kv * dk, dk, dim}, vo{out, heads * dq, dq, dim};
    if (strides != nullptr) {
        View* views[4] = {&vq, &vk, &vv, &vo};
        for (int i = 0; i < 4; ++i) {
            views[i]->b = strides[3 * i];
            views[i]->h = strides[3 * i + 1];
            views[i]->s = strides[3 * i + 2];
        }
    }
    size_t eq, ek, ev, eo;
    if (!strides_ok(vq, batch, heads, seq_q) || !strides_ok(vk, batch, heads_kv, seq_kv) || !strides_ok(vv, batch, heads_kv, seq_kv) ||
        !strides_ok(vo, batch, heads, seq_q) || !extent_of(vq, batch, heads, seq_q, dim, &eq) ||
        !extent_of(vk, batch, heads_kv, seq_kv, dim, &ek) || !extent_of(vv, batch, heads_kv, seq_kv, dim, &ev) ||
        !extent_of(vo, batch, heads, seq_q, dim, &eo) || !rows_apart(vo, batch, heads, seq_q, dim)) {
        return cudaErrorInvalidValue;
    }
    if (host::ranges_overlap(out, eo * 2, q, eq * 2) || host::ranges_overlap(out, eo * 2, k, ek * 2) ||
        host::ranges_overlap(out, eo * 2, v, ev * 2) ||
        (doc_ids != nullptr && host::ranges_overlap(out, eo * 2, doc_ids, static_cast<size_t>(batch) * seq_q * 4)) ||
        (prefix != nullptr && host::ranges_overlap(out, eo * 2, prefix, static_cast<size_t>(batch) * 4)) ||
        (slopes != nullptr && host::ranges_overlap(out, eo * 2, slopes, static_cast<size_t>(heads) * 4))) {
        return cudaErrorInvalidValue;
    }
    int device = 0, sm_count = 0;
    cudaError_t err = host::current_device(&device, &sm_count);
    if (err != cudaSuccess) return err;
    static_cast<void>(cudaGetLastError());

    Params p{};
    p.seq_q = seq_q;
    p.seq_kv = seq_kv;
    p.head_dim = dim;
    // One tile an item where all of them run at once: two tiles share K and V loads and overlap
    // each other's waits, but need more blocks one after the other. 16 heads, causal, 1024 x 128:
    // 22.5 us in pairs, 19.5 one by one.
    const long long all_tiles = bh * ((seq_q + 127LL) / 128);
    p.item_tiles = all_tiles <= sm_count ? 1 : 2;
    p.per_head = p.item_tiles == 1 ? (seq_q + 127) / 128 : pairs;
    p.tile_stride = 2 * pairs;
    p.heads_q = heads;
    p.heads_kv = heads_kv;
    p.group = heads / heads_kv;
    p.num_items = static_cast<int>(bh * p.per_head);
    p.causal = causal;
    p.prefix = prefix;
    p.scale = scale;
    p.scale_log2 = scale * kLog2e;
    p.softcap = softcap;
    p.slopes = slopes;
    p.out = static_cast<uint16_t*>(out);
    p.out_b = vo.b;
    p.out_h = vo.h;
    p.out_s = vo.s;
    p.out_vec = (reinterpret_cast<uintptr_t>(out) & 15u) == 0 && (batch == 1 || vo.b % 8 == 0) && (heads == 1 || vo.h % 8 == 0) &&
                (seq_q == 1 || vo.s % 8 == 0);
    const int grid = p.num_items < sm_count ? p.num_items : sm_count;
    // Items of equal weight go head by head, so that the CTAs running at one time share K and V.
    // Under a causal mask or documents: as many heads as kGroupBytes hold, whole key heads, and at
    // least two items for each SM.
    long long at_once = p.group;
    if (causal != 0 || doc_ids != nullptr) {
        at_once = (kGroupBytes / (4LL * seq_kv * dim)) * p.group;
        const long long fill = (2LL * sm_count + p.per_head - 1) / p.per_head;
        if (at_once < fill) at_once = (fill + p.group - 1) / p.group * p.group;
    }
    p.group_bh = static_cast<int>(at_once < bh ? at_once : bh);

    // One scratch buffer: the item counter, the documents' tiles and rows, copies of
    // operands whose rows TMA cannot address.
    const bool counted = p.num_items > grid;
    const size_t n_tiles = static_cast<size_t>(batch) * 2 * pairs;
    View* in[3] = {&vq, &vk, &vv};
    const int in_heads[3] = {heads, heads_kv, heads_kv}, in_rows[3] = {seq_q, seq_kv, seq_kv};
    size_t bytes = counted ? 256 : 0, tiles_at = 0, rows_at = 0, copy_at[3] = {0, 0, 0};
    auto take = [&](size_t n) {
        const size_t at = bytes;
        bytes += (n + 255) / 256 * 256;
        return at;
    };
    if (doc_ids != nullptr) {
        tiles_at = take(n_tiles * sizeof(int4));
        rows_at = take(static_cast<size_t>(batch) * seq_q * sizeof(int2));
    }
    bool copied[3];
    for (int i = 0; i < 3; ++i) {
        copied[i] = (reinterpret_cast<uintptr_t>(in[i]->p) & 15u) != 0 || (batch > 1 && in[i]->b % 8 != 0) ||
                    (in_heads[i] > 1 && in[i]->h % 8 != 0) || (in_rows[i] > 1 && in[i]->s % 8 != 0);
        if (copied[i]) copy_at[i] = take(static_cast<size_t>(batch) * in_heads[i] * in_rows[i] * dim * 2);
    }
    uint8_t* scratch = nullptr;
    if (bytes > 0) {
        err = host::scratch_alloc(reinterpret_cast<void**>(&scratch), bytes, device, stream);
        if (err != cudaSuccess) return err;
    }
    for (int i = 0; i < 3; ++i) {
        if (!copied[i]) continue;
        const long long rows = in_rows[i], h = in_heads[i];
        uint16_t* dst = reinterpret_cast<uint16_t*>(scratch + copy_at[i]);
        gather_rows_kernel<<<1024, 256, 0, stream>>>(static_cast<const uint16_t*>(in[i]->p), in[i]->b, in[i]->h, in[i]->s, dst,
                                                     in_heads[i], in_rows[i], dim, batch * h * rows * dim);
        *in[i] = View{dst, h * rows * dim, rows * dim, dim};
    }
    if (counted) p.next_item = reinterpret_cast<int*>(scratch);
    if (doc_ids != nullptr) {
        p.tiles = reinterpret_cast<const int4*>(scratch + tiles_at);
        p.rows = reinterpret_cast<const int2*>(scratch + rows_at);
        const dim3 blocks(static_cast<unsigned>((256LL * pairs + kRunThreads - 1) / kRunThreads), static_cast<unsigned>(batch));
        err = host::launch_overlapped(runs_kernel, blocks, kRunThreads, 0, stream, doc_ids, seq_q, 2 * pairs, causal,
                                      reinterpret_cast<int2*>(scratch + rows_at), reinterpret_cast<int4*>(scratch + tiles_at),
                                      p.next_item);
    } else if (counted) {
        err = host::launch_overlapped(zero_kernel, dim3(1), 1, 0, stream, p.next_item);
    }
    CUtensorMap mq, mk, mv;
    if (err != cudaSuccess) {
        // nothing more is launched
    } else if (!(make_map(&mq, vq, batch, heads, seq_q, dim) && make_map(&mk, vk, batch, heads_kv, seq_kv, dim) &&
          make_map(&mv, vv, batch, heads_kv, seq_kv, dim))) {
        err = cudaErrorInvalidValue;
    } else {
        switch ((dim == 128 ? 2 : 0) + (bf16 ? 1 : 0)) {
            case 0: err = launch<64, false>(mq, mk, mv, p, device, grid, stream); break;
            case 1: err = launch<64, true>(mq, mk, mv, p, device, grid, stream); break;
            case 2: err = launch<128, false>(mq, mk, mv, p, device, grid, stream); break;
            default: err = launch<128, true>(mq, mk, mv, p, device, grid, stream); break;
        }
    }
    if (scratch != nullptr) cudaFreeAsync(scratch, stream);
    if (err != cudaSuccess) return err;
    return cudaGetLastError();
}

}  // namespace masked
}  // namespace tk
