// kvcache.cuh — a paged key/value cache held in 8 bits: the plan that gives new
// tokens their places (block tables, slot maps) and the append that quantises
// them into it.
//
// A cache has n_pages pages of `page_size` token places. Page p holds, for each
// key/value head h, a [page_size, head_dim] tile of e4m3 bytes, contiguous, and one
// FP32 scale: a place stands for scale[p, h] * e4m3. Slot s is place s % page_size
// of page s / page_size (64 bits: a cache may hold more than 2^31 places x heads).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <cstdint>

#include "tk_host.cuh"
#include "tk_ptx.cuh"

namespace tk {
namespace kv {

// ---------------------------------------------------------------------------
// e4m3
// ---------------------------------------------------------------------------

// Two FP32 values to two e4m3 bytes (lo in the low byte), nearest even, saturating
// at 448; NaN stays NaN.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Two e4m3 bytes to binary16, exact (subnormals and NaN included).
__device__ __forceinline__ uint32_t from_e4m3x2(uint32_t two) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(two)));
    return r;
}

// Four e4m3 bytes to binary16: bytes 0 and 1 in lo, 2 and 3 in hi.
__device__ __forceinline__ void from_e4m3x4(uint32_t four, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(four));
}

__device__ __forceinline__ float2 half2_bits_to_float2(uint32_t bits) {
    return __half22float2(*reinterpret_cast<const __half2*>(&bits));
}

__device__ __forceinline__ float2 bf162_bits_to_float2(uint32_t bits) {
    return make_float2(__uint_as_float(bits << 16), __uint_as_float(bits & 0xffff0000u));
}

template <bool kBf16>
__device__ __forceinline__ float2 pair_to_float2(uint32_t bits) {
    return kBf16 ? bf162_bits_to_float2(bits) : half2_bits_to_float2(bits);
}

// ---------------------------------------------------------------------------
// Plan
// ---------------------------------------------------------------------------

constexpr int kPlanThreads = 1024;

struct PlanParams {
    const int* cached;   // tokens each request holds in the cache
    const int* fresh;    // tokens it adds now
    int n_requests;
    int page;
    int* table;          // [n_requests, width]
    int width;
    const int* free_pages;
    int free_capacity;
    const int* n_free;
    int* lens_out;       // may be `cached`
    int* seq_lens;
    int* starts;         // [n_requests + 1]
    int64_t* slots;    // [max_tokens]
    int max_tokens;
    int* n_free_out;     // may be `n_free`
};

// Inclusive sum over the CTA's threads (1024), in thread order; `total` gets the sum
// of all. `warp_sums`: 32 values of shared memory.
__device__ __forceinline__ long long block_scan(long long v, long long* warp_sums, long long& total) {
    const int lane = static_cast<int>(lane_id());
    const int warp = static_cast<int>(threadIdx.x >> 5);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    long long w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += up;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const long long before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
    __syncthreads();
    return warp > 0 ? v + before : v;
}

// First index in ends[0, n) (ascending) with ends[i] > x; n if none.
__device__ __forceinline__ int upper_bound(const int* ends, int n, int x) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] > x) hi = mid; else lo = mid + 1;
    }
    return lo;
}

// 1024 requests and what their tokens and pages get, in shared memory.
struct PlanPart {
    int ends[kPlanThreads];   // running new tokens, clamped to INT_MAX
    int upto[kPlanThreads];   // running pages needed, clamped
    int shift[kPlanThreads];  // position of token t of the call: t + shift
    int have[kPlanThreads];   // pages held before
    int base[kPlanThreads];   // number in the call of the page of column c: c + base
    int taken[kPlanThreads];
    long long warp_sums[32];
    int used;                 // pages taken so far
};

__device__ __forceinline__ int clamp_int(long long x) { return static_cast<int>(min(x, static_cast<long long>(INT_MAX))); }

// Table entries and slots of requests r0 .. r0 + here, whose tokens are [tokens, tokens +
// sum) and whose pages [pages, pages + page_sum) of the call, shared out over `ctas` CTAs.
// A warp writes one stretch of consecutive slots, so it searches for its request once, and
// again only where a request ends; four slots a lane are in flight, since each waits for a
// page number from L2.
__device__ __forceinline__ void plan_fill(const PlanParams& p, const PlanPart& part, int r0, int here, long long tokens,
                                          long long sum, long long pages, long long page_sum, int n_free, int rank, int ctas) {
    const int tid = static_cast<int>(threadIdx.x);
    const int lane = static_cast<int>(lane_id());
    const bool pow2 = (p.page & (p.page - 1)) == 0;
    const int shift = 31 - __clz(p.page);
    // Page number k of the call goes to the request whose range holds it.
    const int last_page = static_cast<int>(min(pages + page_sum, static_cast<long long>(n_free)));
    for (long long k = pages + rank * kPlanThreads + tid; k < last_page; k += ctas * kPlanThreads) {
        const int i = upper_bound(part.upto, here, static_cast<int>(k));
        if (i < here && part.taken[i])
            p.table[static_cast<long long>(r0 + i) * p.width + (k - part.base[i])] = p.free_pages[n_free - 1 - k];
    }
    const long long last_token = min(tokens + sum, static_cast<long long>(p.max_tokens));
    const int warps = ctas * (kPlanThreads / 32);
    const long long each = last_token > tokens ? ((last_token - tokens + warps - 1) / warps + 127) / 128 * 128 : 0;
    const long long from = tokens + each * (rank * (kPlanThreads / 32) + (tid >> 5));
    const long long to = min(from + each, last_token);
    int i = from < to ? upper_bound(part.ends, here, static_cast<int>(from)) : 0;
    for (long long t0 = from; t0 < to; t0 += 128) {
        const int first = static_cast<int>(t0), last = static_cast<int>(min(t0 + 128, to)) - 1;
        while (i < here && part.ends[i] <= first) ++i;
        const bool one = i < here && part.ends[i] > last;  // all of them belong to request i
        int owner[4], place[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int t = first + 32 * u + lane;
            owner[u] = -1;
            place[u] = 0;
            if (t > last) continue;
            const int q = one ? i : upper_bound(part.ends, here, t);
            if (q >= here || !part.taken[q]) continue;
            const int pos = t + part.shift[q];
            const int col = pow2 ? pos >> shift : pos / p.page;
            place[u] = pos - col * p.page;
            owner[u] = col < part.have[q] ? p.table[static_cast<long long>(r0 + q) * p.width + col]
                                          : p.free_pages[n_free - 1 - (col + part.base[q])];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int t = first + 32 * u + lane;
            if (t <= last) p.slots[t] = owner[u] >= 0 ? static_cast<long long>(owner[u]) * p.page + place[u] : -1;
        }
    }
}

// Slots behind the last token stand for nothing.
__device__ __forceinline__ void plan_rest(const PlanParams& p, long long tokens, int rank, int ctas) {
    for (long long t = tokens + rank * kPlanThreads + threadIdx.x; t < p.max_tokens; t += ctas * kPlanThreads) p.slots[t] = -1;
}

// Requests 1024 at a time:
//
//   need_r  = ceil((c_r + n_r) / page) - ceil(c_r / page)
//   taken_r = n_r > 0, the row and the slots are wide enough, and need_r = 0 or
//             need_0 + .. + need_r <= n_free
//   page k of the call = free_pages[n_free - 1 - k]
//
// Two prefix sums (new tokens, pages needed), the lengths, and with kFill the entries and
// slots too: then every CTA computes the sums for itself, CTA 0 writes the lengths, and the
// CTAs share out the rest. That needs inputs that CTA 0 does not overwrite. Where lens_out is
// `cached` (a state that moves on in place) and there is more to fill than one CTA should, one
// CTA does the sums without kFill, and plan_fill_kernel follows, which works from that kernel's
// outputs alone, so that no scratch is passed between the two.
// What bounds both: the launches and the chain lengths -> sums -> entries; the bytes are a
// few MB at most (8 a slot). 1024 requests with 385,000 tokens: 39 us when one cluster of
// 8 CTAs did all of it (8 SMs wait for their page numbers), 12.4 us in two kernels, 8.5 in one.
template <bool kFill>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanParams p) {
    __shared__ PlanPart part;
    const int tid = static_cast<int>(threadIdx.x);
    const int rank = static_cast<int>(blockIdx.x), ctas = static_cast<int>(gridDim.x);
    if constexpr (!kFill) grid_release();
    grid_wait();
    int n_free = *p.n_free;
    n_free = n_free < 0 ? 0 : (n_free > p.free_capacity ? p.free_capacity : n_free);
    if (tid == 0) part.used = 0;
    __syncthreads();
    long long tokens = 0, pages = 0;  // sums over the earlier requests
    for (int r0 = 0; r0 < p.n_requests; r0 += kPlanThreads) {
        const int r = r0 + tid;
        int c = 0, n = 0;
        if (r < p.n_requests) {
            c = max(p.cached[r], 0);
            n = max(p.fresh[r], 0);
        }
        long long sum, page_sum;
        const long long end = tokens + block_scan(n, part.warp_sums, sum);
        const long long whole = static_cast<long long>(c) + n;
        const int have = static_cast<int>((static_cast<long long>(c) + p.page - 1) / p.page);
        const bool fits = n > 0 && whole <= min(static_cast<long long>(p.width) * p.page, static_cast<long long>(INT_MAX)) && end <= p.max_tokens;
        const int need = fits ? static_cast<int>((whole + p.page - 1) / p.page) - have : 0;
        const long long upto = pages + block_scan(need, part.warp_sums, page_sum);
        const bool taken = fits && (need == 0 || upto <= n_free);
        if (taken && need > 0) atomicMax(&part.used, static_cast<int>(upto));
        if (rank == 0 && r < p.n_requests) {
            // Each thread has read its own request: with one CTA lens_out may be `cached`.
            p.lens_out[r] = taken ? static_cast<int>(whole) : c;
            p.seq_lens[r] = taken ? static_cast<int>(whole) : 0;
            p.starts[r] = clamp_int(end - n);
        }
        if constexpr (kFill) {
            part.ends[tid] = clamp_int(end);
            part.upto[tid] = clamp_int(upto);
            // Only read where taken: then end <= max_tokens and, if pages are needed, upto <= n_free.
            part.shift[tid] = c - static_cast<int>(end - n);
            part.have[tid] = have;
            part.base[tid] = static_cast<int>(upto - need) - have;
            part.taken[tid] = taken ? 1 : 0;
            __syncthreads();
            plan_fill(p, part, r0, min(kPlanThreads, p.n_requests - r0), tokens, sum, pages, page_sum, n_free, rank, ctas);
            __syncthreads();  // the shared arrays are rewritten by the next 1024 requests
        }
        tokens += sum;
        pages += page_sum;
    }
    __syncthreads();
    if constexpr (kFill) plan_rest(p, tokens, rank, ctas);
    if (rank == 0 && tid == 0) {
        p.starts[p.n_requests] = clamp_int(tokens);
        *p.n_free_out = n_free - part.used;  // may be n_free with one CTA: read at its start
    }
}

// The table entries and slots that follow from plan_kernel's outputs: a request is taken if
// its seq_lens is not 0; then it held lens_out - new tokens. The taken requests that need
// pages are the first ones that do, so the sum of their needs is what n_free went down by.
__global__ void __launch_bounds__(kPlanThreads) plan_fill_kernel(const PlanParams p) {
    __shared__ PlanPart part;
    const int tid = static_cast<int>(threadIdx.x);
    grid_wait();
    // The pages taken in all: free_pages counts from the n_free before the call.
    long long used = 0;
    for (int r0 = 0; r0 < p.n_requests; r0 += kPlanThreads) {
        const int r = r0 + tid;
        int need = 0;
        if (r < p.n_requests && p.seq_lens[r] > 0) {
            const int whole = p.lens_out[r], c = whole - p.fresh[r];
            need = static_cast<int>((static_cast<long long>(whole) + p.page - 1) / p.page - (static_cast<long long>(c) + p.page - 1) / p.page);
        }
        long long page_sum;
        block_scan(need, part.warp_sums, page_sum);
        used += page_sum;
    }
    const int n_free = *p.n_free_out + static_cast<int>(used);
    long long tokens = 0, pages = 0;
    for (int r0 = 0; r0 < p.n_requests; r0 += kPlanThreads) {
        const int r = r0 + tid;
        int c = 0, n = 0, whole = 0;
        bool taken = false;
        long long end = INT_MAX;
        if (r < p.n_requests) {
            n = max(p.fresh[r], 0);
            taken = p.seq_lens[r] > 0;
            whole = p.lens_out[r];
            c = taken ? whole - n : whole;
            end = static_cast<long long>(p.starts[r]) + n;
        }
        const int have = static_cast<int>((static_cast<long long>(c) + p.page - 1) / p.page);
        const int need = taken ? static_cast<int>((static_cast<long long>(whole) + p.page - 1) / p.page) - have : 0;
        long long page_sum;
        const long long upto = pages + block_scan(need, part.warp_sums, page_sum);
        part.ends[tid] = clamp_int(end);
        part.upto[tid] = clamp_int(upto);
        part.shift[tid] = c - static_cast<int>(end - n);
        part.have[tid] = have;
        part.base[tid] = static_cast<int>(upto - need) - have;
        part.taken[tid] = taken ? 1 : 0;
        __syncthreads();
        const int here = min(kPlanThreads, p.n_requests - r0);
        const long long sum = part.ends[here - 1] - tokens;
        plan_fill(p, part, r0, here, tokens, sum, pages, page_sum, n_free, static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x));
        __syncthreads();
        tokens += sum;
        pages += page_sum;
    }
    plan_rest(p, tokens, static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x));
}

inline cudaError_t plan_entry(const int* cached, const int* fresh, int n_requests, int page, int* table, int width,
                              const int* free_pages, int free_capacity, const int* n_free, int* lens_out, int* seq_lens,
                              int* starts, int64_t* slots, int max_tokens, int* n_free_out, cudaStream_t stream) {
    // Arrays without an element may be null.
    const bool none = n_requests == 0;
    if ((!none && (cached == nullptr || fresh == nullptr || lens_out == nullptr || seq_lens == nullptr || table == nullptr)) ||
        n_free == nullptr || starts == nullptr || n_free_out == nullptr || n_requests < 0 || width <= 0 || page <= 0 ||
        free_capacity < 0 || max_tokens < 0 || (free_pages == nullptr && free_capacity > 0) ||
        (slots == nullptr && max_tokens > 0)) {
        return cudaErrorInvalidValue;
    }
    for (const void* p : {static_cast<const void*>(cached), static_cast<const void*>(fresh), static_cast<const void*>(table),
                          static_cast<const void*>(free_pages), static_cast<const void*>(n_free), static_cast<const void*>(lens_out),
                          static_cast<const void*>(seq_lens), static_cast<const void*>(starts), static_cast<const void*>(n_free_out)})
        if (host::misaligned(p, 4)) return cudaErrorInvalidValue;
    if (host::misaligned(slots, 8)) return cudaErrorInvalidValue;
    const size_t bytes = static_cast<size_t>(n_requests) * 4;
    const size_t table_bytes = bytes * static_cast<size_t>(width);
    struct Range { const void* p; size_t n; };
    const Range in[] = {{cached, bytes}, {fresh, bytes}, {free_pages, static_cast<size_t>(free_capacity) * 4}, {n_free, 4}};
    const Range out[] = {{table, table_bytes}, {lens_out, bytes}, {seq_lens, bytes}, {starts, bytes + 4},
                         {slots, static_cast<size_t>(max_tokens) * 8}, {n_free_out, 4}};
    for (int i = 0; i < 6; ++i) {
        for (int j = 0; j < 4; ++j) {
            const bool in_place = (i == 1 && j == 0 && out[i].p == in[j].p) || (i == 5 && j == 3 && out[i].p == in[j].p);
            if (!in_place && host::ranges_overlap(out[i].p, out[i].n, in[j].p, in[j].n)) return cudaErrorInvalidValue;
        }
        for (int j = i + 1; j < 6; ++j)
            if (host::ranges_overlap(out[i].p, out[i].n, out[j].p, out[j].n)) return cudaErrorInvalidValue;
    }
    int sm_count = 0;
    cudaError_t err = host::current_device(nullptr, &sm_count);
    if (err != cudaSuccess) return err;
    static_cast<void>(cudaGetLastError());
    PlanParams p{cached, fresh, n_requests, page, table, width, free_pages, free_capacity, n_free,
                 lens_out, seq_lens, starts, slots, max_tokens, n_free_out};
    // A warp writes 128 slots at a time.
    const long long want = (max_tokens + 4095LL) / 4096;
    const unsigned ctas = static_cast<unsigned>(want < 1 ? 1 : (want < sm_count ? want : sm_count));
    if (ctas == 1 || (lens_out != cached && n_free_out != n_free)) {
        err = host::launch_overlapped(plan_kernel<true>, dim3(ctas), kPlanThreads, 0, stream, p);
        return err != cudaSuccess ? err : cudaGetLastError();
    }
    err = host::launch_overlapped(plan_kernel<false>, dim3(1), kPlanThreads, 0, stream, p);
    if (err == cudaSuccess) err = host::launch_overlapped(plan_fill_kernel, dim3(ctas), kPlanThreads, 0, stream, p);
    return err != cudaSuccess ? err : cudaGetLastError();
}

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------

constexpr int kAppendThreads = 128;
constexpr int kAppendWarps = kAppendThreads / 32;
constexpr int kMostPage = 128;
constexpr int kMostChunk = 64;
constexpr int kLeastExponent = -100;  // of a scale: what is smaller than 2^-109 becomes 0

struct AppendParams {
    const uint16_t* x[2];       // keys, values: [n_tokens, heads, dim], 16-bit
    long long stride[2];        // elements from one token to the next
    const int64_t* slots;
    int n_tokens, heads;
    uint8_t* cache[2];
    float* scale[2];
    long long n_pages;
    int page, page_shift;       // a power of two, and which
    int chunk;                  // tokens per CTA
};

// The smallest power of two s >= 2^kLeastExponent with amax <= 448 s (amax >= 0, finite).
// 448 = 1.75 * 2^8. A power of two costs a floating format no precision, and moving a
// page to a larger scale is then exact but for what falls below e4m3's last step.
__device__ __forceinline__ float scale_for(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    int e = static_cast<int>(bits >> 23) - 127;  // subnormals: -127, below the least anyway
    e = e - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = max(e, kLeastExponent);
    return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// |x| of finite values; infinities and NaN do not set a scale (they are stored as 448
// and NaN).
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.0f;
}

// The larger of each of two 16-bit values; a NaN gives way.
template <bool kBf16>
__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (kBf16) asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Whether neither of two 16-bit magnitudes is infinite or NaN.
template <bool kBf16>
__device__ __forceinline__ bool all_finite(uint32_t pair) {
    constexpr uint32_t inf = kBf16 ? 0x7f80u : 0x7c00u;
    return (pair & 0xffffu) < inf && (pair >> 16) < inf;
}

// |x| of a pair of 16-bit values, 0 for those that are not finite.
template <bool kBf16>
__device__ __forceinline__ uint32_t finite_magnitudes(uint32_t pair) {
    const uint32_t a = pair & 0x7fff7fffu;
    return a & __vcmpltu2(a, kBf16 ? 0x7f807f80u : 0x7c007c00u);
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// a * b rounded to odd: rounded once more, to e4m3's 4 bits, it is the exact product rounded once (a product next to
// a tie of e4m3 would become that tie in FP32).
__device__ __forceinline__ float product_to_odd(float a, float b) {
    const float p = __fmul_rz(a, b);
    return fmaf(a, b, -p) == 0.0f ? p : __uint_as_float(__float_as_uint(p) | 1u);
}

// Whether x * (1 / s) is x / s: s a power of two with a normal reciprocal.
__device__ __forceinline__ bool exact_reciprocal(float s) {
    return (__float_as_uint(s) & 0x7fffffu) == 0 && s >= 7.9e-31f && s < 1.7e38f;
}

// A run is a stretch of consecutive tokens whose slots are consecutive places of one
// page. One warp (or, kCta, the four warps of a CTA together) takes one run of one
// head: the largest |x| of the run sets the scale (never below the page's own, if the
// page already held tokens before the run's first place), the tokens already there move
// to it if it grew, and the run is stored. Grid: (token chunks x heads, keys / values),
// heads fastest: the heads of a token lie side by side, and read at about the same time they
// share DRAM pages. A run belongs to the CTA that holds its first token; it may end behind that CTA's chunk,
// so the CTA looks at one slot before its chunk and a page's worth behind it.
//
// What bounds it: 2 bytes read and 1 written per element; at a few tokens, the chain
// slots -> values -> scale -> bytes (64 tokens x 8 heads x 128: 2.9 us). 28,000 tokens of prompts x 8 x
// 128, pages of 64: 34.4 us = 5.0 TB/s, 77 % of the measured copy bandwidth; each CTA waits for its slots
// before its values, and 8 CTAs an SM (64 registers) cover most of that. A warp for each run
// took 68 us there.
template <int kDim, bool kBf16, bool kCta>
__global__ void __launch_bounds__(kAppendThreads, kCta ? 8 : 1) append_kernel(const AppendParams p) {
    constexpr int kLanes = kDim / 8;                      // threads that read one token, 16 bytes each
    constexpr int kGroup = kCta ? kAppendThreads : 32;    // threads that work on one run
    constexpr int kRows = kGroup / kLanes;                // tokens per step
    constexpr int kHeld = 8;                              // steps held in registers
    __shared__ long long s_slots[1 + kMostChunk + kMostPage];
    __shared__ float s_max[kAppendWarps];
    const bool values = blockIdx.y != 0;
    const int head = static_cast<int>(blockIdx.x) % p.heads;
    const int tid = static_cast<int>(threadIdx.x);
    const int lane = static_cast<int>(lane_id());
    const int warp = tid >> 5;
    const int in_group = kCta ? tid : lane;
    const int t0 = static_cast<int>(blockIdx.x) / p.heads * p.chunk;
    const int count = min(p.chunk, p.n_tokens - t0);
    const uint16_t* x = (values ? p.x[1] : p.x[0]) + head * kDim;
    const long long stride = values ? p.stride[1] : p.stride[0];
    uint8_t* cache = values ? p.cache[1] : p.cache[0];
    float* scales = values ? p.scale[1] : p.scale[0];
    const long long n_slots = p.n_pages * p.page;
    const int sub = in_group / kLanes, col = (in_group % kLanes) * 8;
    grid_wait();

    // s_slots[1 + i]: slot of token t0 + i, -1 where there is no such token or place.
    for (int i = tid; i < 1 + count + p.page; i += kAppendThreads) {
        const long long t = static_cast<long long>(t0) + i - 1;
        long long s = t >= 0 && t < p.n_tokens ? p.slots[t] : -1;
        if (s < 0 || s >= n_slots) s = -1;
        s_slots[i] = s;
    }
    __syncthreads();

    // Every warp finds the first tokens of runs; without kCta it takes every fourth.
    int seen = 0;
    for (int base = 0; base < count; base += 32) {
        const int i = base + lane;
        bool first = false;
        if (i < count) {
            const long long s = s_slots[1 + i], before = s_slots[i];
            first = s >= 0 && (before < 0 || before + 1 != s || (s & (p.page - 1)) == 0);
        }
        uint32_t firsts = __ballot_sync(0xffffffffu, first);
        while (firsts != 0) {
            const int begin = base + __ffs(firsts) - 1;
            firsts &= firsts - 1;
            if (!kCta && (seen++ & (kAppendWarps - 1)) != warp) continue;
            const long long slot = s_slots[1 + begin];
            const int place = static_cast<int>(slot & (p.page - 1));
            // Length of the run: at most to the page's end.
            const int most = p.page - place;
            int n = 1;
            while (n < most) {
                const int j = n + lane;
                const uint32_t mask = __ballot_sync(0xffffffffu, j < most && s_slots[1 + begin + j] == slot + j);
                const int more = mask == 0xffffffffu ? 32 : __ffs(~mask) - 1;
                n += more;
                if (more < 32) break;
            }
            const long long tile = (slot >> p.page_shift) * p.heads + head;
            uint8_t* bytes = cache + tile * p.page * kDim;
            const float old = place > 0 ? scales[tile] : 0.0f;
            const uint16_t* rows = x + static_cast<long long>(t0 + begin) * stride + col;
            uint4 held[kHeld];
            const long long step = kRows * stride;
            auto load = [&](int j0) {
                const uint16_t* at = rows + (j0 + sub) * stride;
                if (j0 + kRows * kHeld <= n) {
#pragma unroll
                    for (int u = 0; u < kHeld; ++u) held[u] = *(reinterpret_cast<const uint4*>(at + u * step));
                } else {
#pragma unroll
                    for (int u = 0; u < kHeld; ++u)
                        held[u] = j0 + u * kRows + sub < n ? *(reinterpret_cast<const uint4*>(at + u * step)) : make_uint4(0, 0, 0, 0);
                }
            };
            // Largest magnitudes of the even and the odd elements.
            uint32_t top = 0;
            for (int j0 = 0; j0 < n; j0 += kRows * kHeld) {
                load(j0);
#pragma unroll
                for (int u = 0; u < kHeld; ++u) {
                    const uint32_t a = max_pair<kBf16>(held[u].x & 0x7fff7fffu, held[u].y & 0x7fff7fffu);
                    const uint32_t b = max_pair<kBf16>(held[u].z & 0x7fff7fffu, held[u].w & 0x7fff7fffu);
                    top = max_pair<kBf16>(top, max_pair<kBf16>(a, b));
                }
            }
            if (__any_sync(0xffffffffu, !all_finite<kBf16>(top))) {
                // Infinities and NaN do not set the scale: once more without them.
                top = 0;
                for (int j0 = 0; j0 < n; j0 += kRows * kHeld) {
                    if (n > kRows * kHeld) load(j0);
#pragma unroll
                    for (int u = 0; u < kHeld; ++u) {
                        const uint32_t w[4] = {held[u].x, held[u].y, held[u].z, held[u].w};
#pragma unroll
                        for (int c = 0; c < 4; ++c) top = max_pair<kBf16>(top, finite_magnitudes<kBf16>(w[c]));
                    }
                }
            }
            const float2 tops = pair_to_float2<kBf16>(top);
            float amax = warp_max(fmaxf(tops.x, tops.y));
            if constexpr (kCta) {
                __syncthreads();  // the last run's maxima have been read, and its scale
                if (lane == 0) s_max[warp] = amax;
                __syncthreads();
                amax = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
            }
            const float now = fmaxf(old, scale_for(amax));
            if (place > 0 && now != old) {
                // The tokens already in the page, to the new scale.
                const float factor = __fdiv_rn(old, now);
                for (int b = in_group * 16; b < place * kDim; b += kGroup * 16) {
                    const uint4 v = *reinterpret_cast<const uint4*>(bytes + b);
                    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float2 lo = half2_bits_to_float2(from_e4m3x2(w[c] & 0xffffu));
                        const float2 hi = half2_bits_to_float2(from_e4m3x2(w[c] >> 16));
                        w[c] = to_e4m3x2(product_to_odd(lo.x, factor), product_to_odd(lo.y, factor)) |
                               to_e4m3x2(product_to_odd(hi.x, factor), product_to_odd(hi.y, factor)) << 16;
                    }
                    *reinterpret_cast<uint4*>(bytes + b) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            auto store = [&](auto over) {
                for (int j0 = 0; j0 < n; j0 += kRows * kHeld) {
                    if (n > kRows * kHeld) load(j0);  // else the registers still hold the run
                    uint8_t* at = bytes + (place + j0 + sub) * kDim + col;
                    const bool full = j0 + kRows * kHeld <= n;
#pragma unroll
                    for (int u = 0; u < kHeld; ++u) {
                        const uint32_t w[4] = {held[u].x, held[u].y, held[u].z, held[u].w};
                        uint32_t b[4];
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float2 f = pair_to_float2<kBf16>(w[c]);
                            b[c] = to_e4m3x2(over(f.x), over(f.y));
                        }
                        if (full || j0 + u * kRows + sub < n)
                            *reinterpret_cast<uint2*>(at + u * kRows * kDim) =
                                make_uint2(__byte_perm(b[0], b[1], 0x5410), __byte_perm(b[2], b[3], 0x5410));
                    }
                }
            };
            if (exact_reciprocal(now)) {
                const float inv = 1.0f / now;
                store([inv](float f) { return f * inv; });
            } else {  // a page's older scale that this library did not choose
                store([now](float f) { return __fdiv_rn(f, now); });
            }
            if (in_group == 0) scales[tile] = now;
        }
    }
}

inline cudaError_t append_entry(bool bf16, const void* k, const void* v, long long k_stride, long long v_stride,
                                const int64_t* slots, int n_tokens, int heads, int dim, void* k_cache, void* v_cache,
                                float* k_scale, float* v_scale, long long n_pages, int page, cudaStream_t stream) {
    if (k == nullptr || v == nullptr || slots == nullptr || k_cache == nullptr || v_cache == nullptr ||
        k_scale == nullptr || v_scale == nullptr || n_tokens < 0 || heads <= 0 || heads > 65535 ||
        (dim != 64 && dim != 128) || n_pages <= 0 || (page != 16 && page != 32 && page != 64 && page != 128)) {
        return cudaErrorInvalidValue;
    }
    const long long row = static_cast<long long>(heads) * dim;
    if (k_stride < row || v_stride < row || k_stride % 8 != 0 || v_stride % 8 != 0 || host::misaligned(k, 16) ||
        host::misaligned(v, 16) || host::misaligned(k_cache, 16) || host::misaligned(v_cache, 16) || host::misaligned(k_scale, 4) ||
        host::misaligned(v_scale, 4) || host::misaligned(slots, 8) ||
        n_pages > LLONG_MAX / page / row || (n_tokens > 0 && (k_stride > LLONG_MAX / 2 / n_tokens || v_stride > LLONG_MAX / 2 / n_tokens))) {
        return cudaErrorInvalidValue;
    }
    const size_t cache_bytes = static_cast<size_t>(n_pages) * page * row, scale_bytes = static_cast<size_t>(n_pages) * heads * 4;
    const size_t x_bytes[2] = {n_tokens > 0 ? (static_cast<size_t>(n_tokens - 1) * k_stride + row) * 2 : 0,
                               n_tokens > 0 ? (static_cast<size_t>(n_tokens - 1) * v_stride + row) * 2 : 0};
    const void* outs[4] = {k_cache, v_cache, k_scale, v_scale};
    const size_t out_bytes[4] = {cache_bytes, cache_bytes, scale_bytes, scale_bytes};
    for (int i = 0; i < 4; ++i) {
        if (host::ranges_overlap(outs[i], out_bytes[i], k, x_bytes[0]) || host::ranges_overlap(outs[i], out_bytes[i], v, x_bytes[1]) ||
            host::ranges_overlap(outs[i], out_bytes[i], slots, static_cast<size_t>(n_tokens) * 8))
            return cudaErrorInvalidValue;
        for (int j = i + 1; j < 4; ++j)
            if (host::ranges_overlap(outs[i], out_bytes[i], outs[j], out_bytes[j])) return cudaErrorInvalidValue;
    }
    cudaError_t err = host::current_device(nullptr, nullptr);
    if (err != cudaSuccess) return err;
    static_cast<void>(cudaGetLastError());
    if (n_tokens == 0) return cudaSuccess;
    AppendParams p{};
    p.x[0] = static_cast<const uint16_t*>(k);
    p.x[1] = static_cast<const uint16_t*>(v);
    p.stride[0] = k_stride;
    p.stride[1] = v_stride;
    p.slots = slots;
    p.n_tokens = n_tokens;
    p.heads = heads;
    p.cache[0] = static_cast<uint8_t*>(k_cache);
    p.cache[1] = static_cast<uint8_t*>(v_cache);
    p.scale[0] = k_scale;
    p.scale[1] = v_scale;
    p.n_pages = n_pages;
    p.page = page;
    p.page_shift = page == 16 ? 4 : (page == 32 ? 5 : (page == 64 ? 6 : 7));
    // Few tokens: each is likely a run of its own (a decode step), one to a warp. Many: runs
    // of up to a page, one at a time by the whole CTA. The number of tokens stands in for the length of
    // the runs, which the host does not know, and errs where few tokens are one prompt or many are single. A warp
    // a run / a CTA a run in chunks of 16 / of 64 tokens, 8 heads of 128, pages of 32, us: 64 single tokens 2.8 / 18.5 /
    // 68, 1024 single 15.8 / 42.7 / 76, 2048 single 29.6 / 78 / 106; one prompt of 256 4.3 / 2.8 / 3.9, of 1024 8.7 / 4.1
    // / 4.3, of 4096 26.5 / 9.7 / 7.6; 8 prompts of 1000 49 / 17.0 / 14.0, 16 of 1000 101 / 33.6 / 26.9.
    const bool cta = n_tokens > 1024;
    p.chunk = cta ? (n_tokens <= 8192 ? 16 : kMostChunk) : kAppendWarps;
    const long long ctas = (n_tokens + p.chunk - 1LL) / p.chunk * heads;
    if (ctas > INT_MAX) return cudaErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(ctas), 2);
    switch ((dim == 128 ? 4 : 0) + (bf16 ? 2 : 0) + (cta ? 1 : 0)) {
        case 0: err = host::launch_overlapped(append_kernel<64, false, false>, grid, kAppendThreads, 0, stream, p); break;
        case 1: err = host::launch_overlapped(append_kernel<64, false, true>, grid, kAppendThreads, 0, stream, p); break;
        case 2: err = host::launch_overlapped(append_kernel<64, true, false>, grid, kAppendThreads, 0, stream, p); break;
        case 3: err = host::launch_overlapped(append_kernel<64, true, true>, grid, kAppendThreads, 0, stream, p); break;
        case 4: err = host::launch_overlapped(append_kernel<128, false, false>, grid, kAppendThreads, 0, stream, p); break;
        case 5: err = host::launch_overlapped(append_kernel<128, false, true>, grid, kAppendThreads, 0, stream, p); break;
        case 6: err = host::launch_overlapped(append_kernel<128, true, false>, grid, kAppendThreads, 0, stream, p); break;
        default: err = host::launch_overlapped(append_kernel<128, true, true>, grid, kAppendThreads, 0, stream, p); break;
    }
    return err != cudaSuccess ? err : cudaGetLastError();
}

}  // namespace kv
}  // namespace tk
