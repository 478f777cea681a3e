// paged_cache.cuh -- a key/value cache in pages shared by a batch of requests: the step's plan
// (block tables and slot maps from the requests' lengths) and the write of new keys and values.
//
// A cache of one layer is [pages][page_size][kv_heads][head_dim] (bf16, fp16, or the engine's int8
// codes with one fp32 scale per 64 dims, [pages][page_size][kv_heads][head_dim / 64]).  Slot s is
// position s % page_size of page s / page_size; a request's block table names its pages in order.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "engine_ops.cuh"

namespace asdsl {

// Division of 0 <= n < 2^31 by a positive int that is fixed for a launch, as a multiply-high
// (Granlund and Montgomery, "Division by invariant integers using multiplication").
struct FastDiv {
    uint32_t mul, shift;
    int d;
    static FastDiv make(int d) {
        FastDiv f;
        f.d = d;
        uint32_t s = 0;
        while ((1ull << s) < static_cast<unsigned long long>(d)) ++s;
        f.shift = s;
        f.mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << s) - static_cast<unsigned long long>(d))) /
                                          static_cast<unsigned long long>(d) +
                                      1);
        return f;
    }
    __device__ __forceinline__ int div(int n) const {
        const uint32_t u = static_cast<uint32_t>(n);
        return static_cast<int>((__umulhi(u, mul) + u) >> shift);
    }
};

// ---------------------------------------------------------------------------
// plan of one step
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 512;
constexpr int kPlanMaxRequests = 12288;  // two int32 prefix sums of the requests in shared memory

enum : int { kPlanFreeShort = 1, kPlanTableNarrow = 2, kPlanTokensOver = 4 };

struct PlanArgs {
    const int32_t* kv_lens;    // [n] tokens each request holds before the step
    const int32_t* new_lens;   // [n] tokens it gains in it
    const int32_t* free_pages; // [n_free] pages nobody holds, taken from the front
    int32_t* table;            // [n][width], row stride table_stride
    int32_t* cu;               // [n + 1]
    int32_t* total;            // [n]
    int32_t* slots;            // [max_tokens]
    int32_t* positions;
    int32_t* requests;
    int32_t* counts;           // pages needed, tokens, flags
    long long table_stride;
    int n, n_free, width, max_tokens;
    FastDiv page;
};

__device__ __forceinline__ int sat_add(int a, int b) {  // a, b >= 0
    const uint32_t s = static_cast<uint32_t>(a) + static_cast<uint32_t>(b);
    return s > 0x7fffffffu ? 0x7fffffff : static_cast<int>(s);
}

// pages that hold n tokens, at most the table's width (n may be INT_MAX)
__device__ __forceinline__ int pages_for(int n, const PlanArgs& a) {
    const int p = n <= 0 ? 0 : a.page.div(n - 1) + 1;
    return p < a.width ? p : a.width;
}

// index of the last entry of the ascending pre[0..n] that is <= x (pre[0] = 0 <= x < pre[n])
__device__ __forceinline__ int last_not_above(const int32_t* pre, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Every CTA computes the two prefix sums over the requests (tokens and new pages) for itself in
// shared memory and then fills its share of the tokens and of the new table cells, so the step's
// whole plan is one launch without a grid-wide wait.  Saturating sums keep lengths that add up past
// int32 ordered.  A slot in a page the request held before is read from the table (cells below the
// old page count, which this kernel never writes); a slot in a new page from the free list.
__global__ void __launch_bounds__(kPlanThreads) k_plan_step(const PlanArgs a) {
    extern __shared__ int32_t plan_smem[];
    int32_t* cu = plan_smem;              // [n + 1]
    int32_t* po = plan_smem + a.n + 1;    // [n + 1]
    __shared__ int warp_tok[kPlanThreads / 32], warp_pg[kPlanThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        cu[0] = 0;
        po[0] = 0;
    }
    int tok_base = 0, pg_base = 0;
    bool outgrown = false;
    for (int r0 = 0; r0 < a.n; r0 += kPlanThreads) {
        const int r = r0 + tid;
        int tok = 0, pg = 0;
        if (r < a.n) {
            const int kv = max(a.kv_lens[r], 0);
            tok = max(a.new_lens[r], 0);
            const int total = sat_add(kv, tok);
            pg = pages_for(total, a) - pages_for(kv, a);
            if (blockIdx.x == 0) {
                a.total[r] = total;
                if (tok > 0 && a.page.div(total - 1) >= a.width) outgrown = true;
            }
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, tok, o), p = __shfl_up_sync(0xffffffffu, pg, o);
            if (lane >= o) {
                tok = sat_add(tok, t);
                pg = sat_add(pg, p);
            }
        }
        if (lane == 31) {
            warp_tok[warp] = tok;
            warp_pg[warp] = pg;
        }
        __syncthreads();
        int tb = tok_base, pb = pg_base, ta = tok_base, pa = pg_base;
#pragma unroll
        for (int w = 0; w < kPlanThreads / 32; ++w) {
            if (w == warp) {
                tb = ta;
                pb = pa;
            }
            ta = sat_add(ta, warp_tok[w]);
            pa = sat_add(pa, warp_pg[w]);
        }
        if (r < a.n) {
            cu[r + 1] = sat_add(tb, tok);
            po[r + 1] = sat_add(pb, pg);
        }
        tok_base = ta;
        pg_base = pa;
        __syncthreads();
    }
    const bool narrow = __syncthreads_or(outgrown);
    const int total_tok = tok_base, total_pg = pg_base;
    if (blockIdx.x == 0) {
        for (int r = tid; r <= a.n; r += kPlanThreads) a.cu[r] = cu[r];
        if (tid == 0) {
            a.counts[0] = total_pg;
            a.counts[1] = total_tok;
            a.counts[2] = (total_pg > a.n_free ? kPlanFreeShort : 0) | (narrow ? kPlanTableNarrow : 0) |
                          (total_tok > a.max_tokens ? kPlanTokensOver : 0);
        }
    }
    const int stride = gridDim.x * kPlanThreads, first = blockIdx.x * kPlanThreads + tid;
    // new table cells (past the free list's end: -1)
    for (int j = first; j < total_pg && j >= 0; j += stride) {
        const int r = last_not_above(po, a.n, j);
        const int held = pages_for(max(a.kv_lens[r], 0), a);
        a.table[r * a.table_stride + held + (j - po[r])] = j < a.n_free ? a.free_pages[j] : -1;
    }
    for (int t = first; t < a.max_tokens && t >= 0; t += stride) {
        int slot = -1, pos = 0, req = -1;
        if (t < total_tok) {
            req = last_not_above(cu, a.n, t);
            const int kv = max(a.kv_lens[req], 0);
            pos = sat_add(kv, t - cu[req]);
            const int blk = a.page.div(pos);
            if (blk < a.width) {
                const int held = pages_for(kv, a);
                int pg = -1;
                if (blk < held) {
                    pg = a.table[req * a.table_stride + blk];
                } else {
                    const int j = sat_add(po[req], blk - held);
                    if (j < a.n_free) pg = a.free_pages[j];
                }
                const long long s = static_cast<long long>(pg) * a.page.d + (pos - blk * a.page.d);
                if (pg >= 0 && s <= 0x7fffffffll) slot = static_cast<int>(s);
            }
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
        a.requests[t] = req;
    }
}

// ---------------------------------------------------------------------------
// write of new keys and values
// ---------------------------------------------------------------------------
struct CacheView {
    void* k;
    void* v;
    float* ks;  // int8 caches: [pages][page_size][kv_heads][head_dim / 64]
    float* vs;
    long long page_stride, token_stride, head_stride;  // elements
    int n_pages, kv_heads;
    FastDiv page;
};

struct KvWriteArgs {
    const void* k;
    const void* v;
    long long token_stride, head_stride;  // of k and v, elements
    const int32_t* slots;                 // [tokens]; a slot outside the cache is skipped
    CacheView c;
    long long items;                      // tokens * kv_heads * head_dim / 8
    int tokens, head_dim;
    FastDiv heads;  // by kv_heads
};

// eight consecutive elements as fp32
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float2 f;
            if constexpr (std::is_same<T, __half>::value) f = half2_bits_to_float2(w[i]);
            else f = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
}

// two fp32 rounded to nearest even into a 16-bit pair (low half = lo)
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value)
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// One thread per 8 dims of a (token, head), K and V both: 16-byte loads and stores (8-byte code
// stores for int8).  int8: per 64 dims (8 threads) scale = amax * fl(1/127), code = rne(x * inv) clamped to
// +-127, scale 1e-12 for a block of zeros.  The scales are the decode engine's bit for bit; inv is 127 * (1 /
// amax), rounded twice, where the engine rounds 127 / amax once, so a value within 2^-22 of a rounding boundary can
// have the neighbouring code (1.3e-6 of fp32 values; of bf16 ones 3.2e-4, all exact ties).  The values held
// are as near either way (relative error 0.0059301 of normal values, at most 0.50001 steps).
// Bound by memory: 16384 tokens x 8 x 128 bf16 24.6 us (5.5 TB/s), fp32 -> int8 30.9, bf16 -> int8 24.6.
template <typename SRC, typename DST>
__global__ void __launch_bounds__(256) k_kv_write(const KvWriteArgs a) {
    const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    const int shift = a.head_dim == 128 ? 4 : 3;  // threads of a head
    const bool live = i < a.items;  // items is a multiple of 8: the 8 threads of a block agree
    const int th = live ? static_cast<int>(i >> shift) : 0;
    const int d = live ? static_cast<int>(i & ((1 << shift) - 1)) * 8 : 0;
    const int tok = a.heads.div(th), h = th - tok * a.c.kv_heads;
    const int slot = live ? a.slots[tok] : -1;
    const int pg = slot >= 0 ? a.c.page.div(slot) : 0;
    const bool ok = slot >= 0 && pg < a.c.n_pages;
    const int off = slot - pg * a.c.page.d;
    const long long src = static_cast<long long>(tok) * a.token_stride + static_cast<long long>(h) * a.head_stride + d;
    const long long dst = pg * a.c.page_stride + off * a.c.token_stride + h * a.c.head_stride + d;
    // both loads before the first store (the compiler cannot know that the cache is not the source)
    constexpr int NW = sizeof(SRC) * 8 / 16;  // 16-byte words of 8 elements
    uint4 raw[2][NW];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv)
#pragma unroll
        for (int w = 0; w < NW; ++w)
            raw[kv][w] = ok ? __ldg(reinterpret_cast<const uint4*>(static_cast<const SRC*>(kv ? a.v : a.k) + src) + w)
                            : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        DST* o = static_cast<DST*>(kv ? a.c.v : a.c.k) + dst;
        if constexpr (std::is_same<SRC, DST>::value) {
            if (ok) *reinterpret_cast<uint4*>(o) = raw[kv][0];
        } else {
            float x[8];
            load8(reinterpret_cast<const SRC*>(raw[kv]), x);
            if constexpr (sizeof(DST) == 1) {
                float amax = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[e]));
#pragma unroll
                for (int sh = 4; sh > 0; sh >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, sh));
                // the engine's 127 / amax as 127 * (1 / amax), the form of an elementwise program
                const float inv = amax > 1e-12f ? __fmul_rn(127.0f, __frcp_rn(amax)) : __int_as_float(0x5368D4A5);
                uint32_t w[2] = {0, 0};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    int q = __float2int_rn(__fmul_rn(x[e], inv));
                    q = q < -127 ? -127 : (q > 127 ? 127 : q);
                    w[e >> 2] |= (static_cast<uint32_t>(q) & 0xffu) << ((e & 3) * 8);
                }
                if (ok) {
                    *reinterpret_cast<uint2*>(o) = make_uint2(w[0], w[1]);
                    if ((threadIdx.x & 7) == 0) {
                        const long long sb = (static_cast<long long>(slot) * a.c.kv_heads + h) * (a.head_dim >> 6) + (d >> 6);
                        (kv ? a.c.vs : a.c.ks)[sb] = amax > 1e-12f ? __fmul_rn(amax, inv127f()) : 1e-12f;
                    }
                }
            } else {
                if (ok)
                    *reinterpret_cast<uint4*>(o) = make_uint4(pack2<DST>(x[0], x[1]), pack2<DST>(x[2], x[3]),
                                                              pack2<DST>(x[4], x[5]), pack2<DST>(x[6], x[7]));
            }
        }
    }
}

}  // namespace asdsl
