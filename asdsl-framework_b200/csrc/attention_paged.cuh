// attention_paged.cuh -- attention of a batch over a paged cache: few query rows per request.
//
// Row i of a request with n new tokens and len cached ones (the new ones among them) stands at
// position p = len - n + i and sees the keys j <= p with j > p - window or j < sinks.  Keys that no
// row of a tile can see are left out by renumbering: with lo = max(0, p_first - window + 1) the
// tile's keys are the virtual indices 0 .. min(sinks, lo) + (p_last + 1 - lo) - 1, so sinks and
// window are one contiguous run and no tile straddles the gap between them.
//
//   out = sum_j exp(s_j - M) v_j / sum_j exp(s_j - M),  s_j = scale * q . k_j,  M = running maximum
//
// in one pass over the keys, the maximum and sum in fp32; P is rounded to the query's 16-bit type for
// the second product (half a unit in the last place of each weight, as of the output itself), the sum is of the
// unrounded weights.  bf16 has fp32's range; fp16 weights are lifted by a power of two (kLift: M stands that much
// below the maximum, which the quotient does not see), since a long tail of keys can carry the output although
// each of its weights is far below the largest: with weights up to 1, those below 2^-14 of it lost bits and those
// below 2^-25 counted in the sum alone.  Lifted, a weight keeps all its bits down to 2^-29 of the largest (int8
// pages: 2^-28, times its V scale over the block's largest so far; the many-rows kernel 2^-26 and 2^-25).
#pragma once

#include <type_traits>

#include "paged_cache.cuh"

namespace asdsl {

struct AttnPagedArgs {
    const void* q;  // [tokens][heads][head_dim], strides in elements
    long long q_token_stride, q_head_stride;
    CacheView c;
    const int32_t* table;  // [n_req][width], row stride table_stride
    long long table_stride;
    int width;
    const int32_t* lens;  // [n_req]; null: one request of all rows and const_len keys
    int const_len;
    const int32_t* cu;    // [n_req + 1] row starts in q; null: one row per request
    int n_req, tokens, heads, group;
    int causal, window, sinks;
    float scale_log2;
    void* out;  // [tokens][heads][head_dim] contiguous, the query's type
    float* lse; // [tokens][heads] or null
    // Rows joined from parts (unnormalised output, maximum in log2 units, sum): set, an attention launch
    // leaves its part of each of its rows here (part `split`, of the few-rows kernel part 0), and
    // k_attention_join reads n_parts of them.  acc [parts][tokens * heads][head_dim], ml [parts][tokens * heads].
    float* parts_acc;
    float2* parts_ml;
    int n_parts;
    int splits;               // key splits of the many-rows kernel, and of a last block of one row tile
    int splits_last;          // (0: as the others)
    FastDiv by_group;
    int small_rows;           // requests with up to this many rows (tokens x group) go to the few-rows kernel
    float* part;              // partial results of keys split over CTAs
    unsigned int* count;      // [n_req][kv_heads] arrivals per unit, zero before and after a launch
};

constexpr float kLn2 = 0.693147180559945309f;

// ---- one request's share -------------------------------------------------------------------
struct ReqRows {
    int first, n, len;  // first row in q, rows (tokens), keys
    int held;           // of those keys, what the table has cells for: the others are unseen
};

__device__ __forceinline__ ReqRows request_rows(const AttnPagedArgs& a, int b) {
    ReqRows r;
    if (!a.lens) {
        r.first = 0;
        r.n = a.tokens;
    } else if (a.cu) {
        const int c0 = min(max(a.cu[b], 0), a.tokens), c1 = min(max(a.cu[b + 1], 0), a.tokens);
        r.first = c0;
        r.n = max(c1 - c0, 0);
    } else {
        r.first = b;
        r.n = b < a.tokens ? 1 : 0;
    }
    const long long cap = static_cast<long long>(a.width) * a.c.page.d;
    r.len = max(a.lens ? a.lens[b] : a.const_len, 0);
    r.held = r.len < cap ? r.len : static_cast<int>(cap);
    return r;
}

// the keys that rows [i0, i1) of a request can see, as virtual indices
struct KeySpan {
    int lo, sunk, n;  // first key of the window part, sink keys before it, keys in all
    __device__ __forceinline__ int key(int u) const { return u < sunk ? u : lo + (u - sunk); }
};

// first key of the window of a row at position p (p + 1 - window would leave 32 bits for rows before key 0)
__device__ __forceinline__ int window_low(const AttnPagedArgs& a, int p) { return p < a.window ? 0 : p - a.window + 1; }

__device__ __forceinline__ KeySpan key_span(const AttnPagedArgs& a, const ReqRows& r, int i0, int i1) {
    KeySpan s{0, 0, r.held};
    if (a.causal) {
        const int hi = min(max(r.len - r.n + i1, 0), r.held);
        s.n = hi;
        if (a.window > 0) {
            s.lo = min(window_low(a, r.len - r.n + i0), hi);
            s.sunk = min(a.sinks, s.lo);
            s.n = s.sunk + hi - s.lo;
        }
    }
    return s;
}

__device__ __forceinline__ bool row_sees(const AttnPagedArgs& a, int p, int j) {
    return j <= p && (a.window <= 0 || j >= window_low(a, p) || j < a.sinks);
}

// ---- 16-bit tensor-core product ------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 8x8 transpose of 16-bit elements over the warp: lane (g, c) gives (g; 2c, 2c + 1), gets (2c, 2c + 1; g)
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Four int8 codes as two fp16 pairs, exact, by a known method: the byte c + 128 goes into the mantissa of
// 1024 + (c + 128), and 1152 is subtracted.
__device__ __forceinline__ void codes_to_pairs(uint32_t w, uint32_t& p01, uint32_t& p23) {
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    uint32_t x0 = __byte_perm(u, 0x64646464u, 0x4140), x1 = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 r0 = __hsub2(*reinterpret_cast<__half2*>(&x0), off), r1 = __hsub2(*reinterpret_cast<__half2*>(&x1), off);
    p01 = *reinterpret_cast<const uint32_t*>(&r0);
    p23 = *reinterpret_cast<const uint32_t*>(&r1);
}

// asynchronous copies global -> shared of N bytes, of which `bytes` (0 or N) are read and the rest zero
template <int N>
__device__ __forceinline__ void cp_async_n(uint32_t dst, const void* src, int bytes) {
    if constexpr (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A finished piece of a row (DP dims from d0; mx in log2 units, acc and sum relative to it): divided by the
// sum and written, or kept as a part.  A row that saw no key
// (sum 0) gives 0 and a log sum of -inf.
template <typename T, int DP>
__device__ __forceinline__ void attention_store(const AttnPagedArgs& a, int part, long long qh, int D, int d0, bool leads,
                                                float (&acc)[DP], float mx, float sum, bool last = false) {
    if (a.parts_acc && !last) {
        const long long rows = static_cast<long long>(a.tokens) * a.heads;
        float* op = a.parts_acc + (part * rows + qh) * D + d0;
#pragma unroll
        for (int d = 0; d < DP; d += 4) *reinterpret_cast<float4*>(op + d) = make_float4(acc[d], acc[d + 1], acc[d + 2], acc[d + 3]);
        if (leads) a.parts_ml[part * rows + qh] = make_float2(mx, sum);
        return;
    }
    if (leads && a.lse) a.lse[qh] = sum == 0.0f ? -INFINITY : (mx + log2f(sum)) * kLn2;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int d = 0; d < DP; ++d) acc[d] = sum == 0.0f ? 0.0f : acc[d] * inv;
    T* op = static_cast<T*>(a.out) + qh * D + d0;
#pragma unroll
    for (int d = 0; d < DP; d += 8)
        *reinterpret_cast<uint4*>(op + d) = make_uint4(pack2<T>(acc[d], acc[d + 1]), pack2<T>(acc[d + 2], acc[d + 3]),
                                                       pack2<T>(acc[d + 4], acc[d + 5]), pack2<T>(acc[d + 6], acc[d + 7]));
}

// ---- geometry of the few-rows kernel -------------------------------------------------------
// While the work line gives a CTA less than kRowsLong iterations, a unit of up to kRowsWhole of them is not
// split (joining the parts costs more than its keys), longer ones are cut every second iteration.
constexpr int kRowsLong = 4, kRowsWhole = 4;

template <bool I8, int D>
struct RowsGeom {
    static constexpr int kRow = D * (I8 ? 1 : 2);           // bytes of a key
    static constexpr int kKv = 16 * kRow;                   // bytes of a warp's 16 keys (K or V)
    // A warp's keys in shared memory: lines of 128 bytes (half a 256-byte row, a row, or two 64-byte
    // rows) in pieces of 16, permuted within the line so that neither the copies (whole lines) nor the
    // reads of fragments (keys g, piece c; keys 2 c, piece g) conflict.
    static constexpr int kHalves = kRow > 128 ? 2 : 1;
    static constexpr int kEight = kRow < 128 ? 512 : 1024;  // from key k to k + 8
    __device__ static __forceinline__ uint32_t k_at(int key, int piece) {
        if constexpr (kRow < 128) return (key >> 1) * 128 + (((key & 1) * 4 + piece) << 4);
        else return key * 128 + ((piece ^ ((key & 1) << 2)) << 4);
    }
    __device__ static __forceinline__ uint32_t v_at(int key, int piece) {
        if constexpr (kRow < 128) return (key >> 1) * 128 + ((((key & 1) * 4 + piece) ^ ((key >> 1 & 3) << 1)) << 4);
        else return key * 128 + ((piece ^ ((key >> 1 & 3) << 1)) << 4);
    }
    static constexpr int kScale = I8 ? 32 * (D / 64) * 4 : 0;
    static constexpr int kStage = 2 * kKv + kScale;
    static constexpr int kCtas = I8 ? 4 : 3;                // per SM, what the registers allow
    static constexpr int kWarps = 4;
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kTile = 16 * kWarps;               // keys of one iteration: 16 per warp
    static constexpr int kStages = (I8 ? 8 : 16) * 1024 / (2 * kKv);
    static constexpr int kOffsets = 32 * 8;                 // the key offsets of two iterations, from lane to lanes
    static constexpr int kWarp = (kStages * kStage + kOffsets + 4 * kStages + 127) / 128 * 128;
    static constexpr int kRing = kWarps * kWarp;
    static constexpr int kMergeRow = D + 4;
    static constexpr int kMerge = kWarps * 16 * (kMergeRow + 2) * 4;  // the warps' results; then the parts' weights
    static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
};

constexpr int kRowsMaxCtas = 4;

__host__ __device__ constexpr int part_floats(int rows, int D) { return rows * (D + 2); }

// ---- the few-rows kernel -------------------------------------------------------------------
// A unit is a request and KV head: the query rows (group heads times tokens) are one tile of up to 8 NR, which
// the launch rule sees to.  Its keys come in iterations of 16 to each of the 4 warps, which keep their own
// maximum, sum and output.  All units' iterations form one line that is cut into equal runs, one per CTA, so
// the work is even whatever the requests' lengths; a unit cut by a run's end leaves (max, sum, output)
// partials that the last CTA to arrive merges in CTA order (same bits every time).
//
// Both products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that the 16-high side of the
// tensor-core tile is keys (then dims) and the 8-wide side the few rows: half the products, registers and
// exponentials of the other way round, which was held up by its own latencies at 8 warps per SM
// (24 requests x 7k bf16 keys: 157 us, 4.2 TB/s).  P^T goes from accumulator to operand form with one 8x8
// transpose per 8 keys.
//
// Bound by the cache's bytes.  A warp copies whole 128-byte lines of its keys, with cp.async, into its own
// ring in shared memory (16 KB in flight per warp, 8 KB for int8; no block-wide barriers) and reads them back as operand
// fragments: the contraction index of S and the dims of O are permuted so that a lane's fragments are
// 16 consecutive bytes of a key's row.  Copies of 64-byte half lines, each lane its own fragments, had
// the L2's tag lookups at 61 % and held the kernel at 4.5 TB/s.
template <typename T, bool I8, int D, int NR>
__global__ void __launch_bounds__(RowsGeom<I8, D>::kThreads, RowsGeom<I8, D>::kCtas) k_attention_rows_paged(const AttnPagedArgs a) {
    using G = RowsGeom<I8, D>;
    constexpr int NB = D / 64;          // 64-dim blocks
    constexpr int NK = G::kRow / 64;    // 16-byte K pieces per lane and key
    constexpr int kLanes = G::kRow < 128 ? 4 : 8, kGroup = 32 / kLanes;  // lanes of a row, rows of a copy
    constexpr int ES = I8 ? 1 : 2;
    using C = std::conditional_t<I8, __half, T>;  // operand type of the products
    // log2 of the largest weight: below fp16's 65504 (int8: times a V scale over its unit, below 2)
    constexpr float kLift = !std::is_same<C, __half>::value ? 0.0f : (I8 ? 14.0f : 15.0f);
    extern __shared__ __align__(128) uint8_t rows_smem[];
    __shared__ long long s_scan[2][G::kWarps], s_base;
    __shared__ int s_req, s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int kv_heads = a.c.kv_heads;

    // iterations of a request's units (0: no rows, or more than this kernel takes)
    auto iters_of = [&](const ReqRows& r) {
        const int rows = r.n * a.group;
        return rows == 0 || rows > a.small_rows ? 0 : max((key_span(a, r, 0, r.n).n + G::kTile - 1) / G::kTile, 1);
    };
    // The length of the line, in iterations and in chunks; then the request of this CTA's first chunk.  A
    // second pass over the requests is needed only where there are more of them than threads.
    long long total = 0, begin = 0, end = 0;
    int active = 0, chunk = 1;
    const bool once = a.n_req <= G::kThreads;
    for (int pass = 0; pass < 2; ++pass) {
        long long base[2] = {0, 0};
        for (int r0 = 0; r0 < a.n_req; r0 += G::kThreads) {
            const int iters = r0 + tid < a.n_req ? iters_of(request_rows(a, r0 + tid)) : 0;
            const long long cnt[2] = {static_cast<long long>(kv_heads) * iters,
                                      static_cast<long long>(kv_heads) * (iters <= kRowsWhole ? min(iters, 1) : (iters + 1) / 2)};
            long long inc[2] = {cnt[0], cnt[1]};
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long t0 = __shfl_up_sync(0xffffffffu, inc[0], o), t1 = __shfl_up_sync(0xffffffffu, inc[1], o);
                if (lane >= o) {
                    inc[0] += t0;
                    inc[1] += t1;
                }
            }
            if (lane == 31) {
                s_scan[0][warp] = inc[0];
                s_scan[1][warp] = inc[1];
            }
            __syncthreads();
            long long before[2] = {base[0], base[1]};
#pragma unroll
            for (int w = 0; w < G::kWarps; ++w) {
                if (w < warp) {
                    before[0] += s_scan[0][w];
                    before[1] += s_scan[1][w];
                }
                base[0] += s_scan[0][w];
                base[1] += s_scan[1][w];
            }
            if (once) {
                chunk = base[0] < static_cast<long long>(kRowsLong) * gridDim.x ? 2 : 1;
                total = chunk > 1 ? base[1] : base[0];
                active = total < gridDim.x ? static_cast<int>(total) : static_cast<int>(gridDim.x);
                begin = total * blockIdx.x / max(active, 1);
            }
            if (once || pass == 1) {
                const int k = chunk > 1 ? 1 : 0;
                const long long n = k ? cnt[1] : cnt[0], mine = k ? before[1] + inc[1] - n : before[0] + inc[0] - n;
                if (n > 0 && mine <= begin && begin < mine + n) {
                    s_req = r0 + tid;
                    s_base = mine;
                }
            }
            __syncthreads();
        }
        if (pass == 0) {
            chunk = base[0] < static_cast<long long>(kRowsLong) * gridDim.x ? 2 : 1;
            total = chunk > 1 ? base[1] : base[0];
            active = total < gridDim.x ? static_cast<int>(total) : static_cast<int>(gridDim.x);
            if (static_cast<int>(blockIdx.x) >= active) return;
            begin = total * blockIdx.x / active;
            end = total * (blockIdx.x + 1) / active;
            if (once) break;
        }
    }
    int req = s_req;
    long long req_base = s_base;
    auto chunks_of = [&](int iters) { return chunk == 1 ? iters : (iters <= kRowsWhole ? min(iters, 1) : (iters + 1) / 2); };
    auto start_of = [&](int cta) { return total * cta / active; };
    auto cta_of = [&](long long y) { return static_cast<int>(((y + 1) * active - 1) / total); };  // last with start <= y

    const uint32_t ring = smem_u32(rows_smem) + warp * G::kWarp, offs = ring + G::kStages * G::kStage,
                   haves = offs + G::kOffsets;  // per stage: which of its 16 keys exist
    for (long long x = begin; x < end;) {
        ReqRows r = request_rows(a, req);
        int iters = iters_of(r), chunks = chunks_of(iters);
        while (x >= req_base + static_cast<long long>(kv_heads) * chunks) {
            req_base += static_cast<long long>(kv_heads) * chunks;
            ++req;
            r = request_rows(a, req);
            iters = iters_of(r);
            chunks = chunks_of(iters);
        }
        const int h = static_cast<int>((x - req_base) / chunks);
        const long long unit_x = req_base + static_cast<long long>(h) * chunks;
        const int c0 = static_cast<int>(x - unit_x), c1 = static_cast<int>(min(end - unit_x, static_cast<long long>(chunks)));
        const int it0 = c0 * chunk, it1 = c1 == chunks ? iters : c1 * chunk;
        const int rows = r.n * a.group;
        const KeySpan span = key_span(a, r, 0, r.n);
        const bool same = !a.causal || r.n == 1;  // all rows see all of the span

        // page of this lane's key, of iteration `it` (lanes 0-15) or the next (16-31); -1: no such key
        const int32_t* tab = a.table + req * a.table_stride;
        const int my_u = (lane >> 4) * G::kTile + warp * 16 + (lane & 15);
        auto lookup = [&](int it) {
            const int u = it * G::kTile + my_u;
            if (it + (lane >> 4) >= it1 || u >= span.n) return -1;
            const int pg = tab[a.c.page.div(span.key(u))];
            return pg < a.c.n_pages ? pg : -1;
        };
        const int piece = lane % kLanes, sub = lane / kLanes;  // this lane's 16 bytes of a row, its row of a group
        const char* kp = static_cast<const char*>(a.c.k) + static_cast<long long>(h) * a.c.head_stride * ES + 16 * piece;
        const char* vp = static_cast<const char*>(a.c.v) + static_cast<long long>(h) * a.c.head_stride * ES + 16 * piece;
        // the byte offsets of the keys of iterations it and it + 1, for all lanes; odd where there is no such key (its pieces are filled with zeros)
        long long scale_at = 0;  // int8: where this lane's key has its scales
        uint32_t have = 0;
        auto prepare = [&](int it, int pg) {
            const bool ok = pg >= 0;
            const int j = span.key(it * G::kTile + my_u);
            const int in_page = ok ? j - a.c.page.div(j) * a.c.page.d : 0;
            const long long off = ok ? (pg * a.c.page_stride + in_page * a.c.token_stride) * ES : 1;
            have = __ballot_sync(0xffffffffu, ok);
            if constexpr (I8) scale_at = ok ? ((static_cast<long long>(pg) * a.c.page.d + in_page) * kv_heads + h) * NB : -1;
            __syncwarp();  // the offsets before these are read
            asm volatile("st.shared.b64 [%0], %1;" ::"r"(offs + lane * 8), "l"(off) : "memory");
            __syncwarp();
        };
        auto issue = [&](int slot, int odd) {
            const uint32_t st = ring + slot * G::kStage, of = offs + odd * 128;
#pragma unroll
            for (int j = 0; j < 16 / kGroup; ++j) {
                const int key = kGroup * j + sub;
                const uint2 o = lds64(of + key * 8);
                const int bytes = o.x & 1u ? 0 : 16;
                const long long off = static_cast<long long>(static_cast<unsigned long long>(o.y) << 32 | (o.x & ~1u));
                const uint32_t dk = st + G::k_at(key, piece), dv = st + G::kKv + G::v_at(key, piece);
#pragma unroll
                for (int b = 0; b < G::kHalves; ++b) {
                    cp_async_n<16>(dk + b * 2048, kp + off + b * 128, bytes);
                    cp_async_n<16>(dv + b * 2048, vp + off + b * 128, bytes);
                }
            }
            if constexpr (I8) {
                // lanes 0-15 the K scales, 16-31 the V scales
                const long long sb = __shfl_sync(0xffffffffu, scale_at, 16 * odd + (lane & 15));
                cp_async_n<4 * NB>(st + 2 * G::kKv + lane * 4 * NB, (lane < 16 ? a.c.ks : a.c.vs) + (sb < 0 ? 0 : sb), sb < 0 ? 0 : 4 * NB);
            }
            if (lane == 0) asm volatile("st.shared.b32 [%0], %1;" ::"r"(haves + slot * 4), "r"(have >> (16 * odd) & 0xffffu) : "memory");
        };

        // where this lane's fragments lie in a stage: K of key g, pieces c and c + 4; V of keys 2 c and
        // 2 c + 1, dims 8 g .. (16-bit: of each half; int8: of each 64-dim block)
        const uint32_t k_read[2] = {G::k_at(g, c), G::kRow < 128 ? 0u : G::k_at(g, c + 4)};
        uint32_t v_read[I8 ? NB : 1][2];
#pragma unroll
        for (int i = 0; i < (I8 ? NB : 1); ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                v_read[i][e] = G::kKv + (I8 ? G::v_at(2 * c + e, 4 * i + (g >> 1)) + 8 * (g & 1) : G::v_at(2 * c + e, g));

        int pg = lookup(it0), slot = 0;
#pragma unroll
        for (int s = 0; s < G::kStages; ++s) {
            if (s % 2 == 0) {
                prepare(it0 + s, pg);
                pg = lookup(it0 + s + 2);
            }
            issue(s, s % 2);
            cp_async_commit();
        }

        // ---- query fragments: row g of each 8, in the order of the K pieces ----
        constexpr int NQ = D / 32;
        uint4 qf[NR][NQ];
        float q_scale[NR][2];  // log2 units of a score of rows 2 c and 2 c + 1
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const int row = g + 8 * n, i = row / a.group;
            const bool live = row < rows;
            const T* qp = static_cast<const T*>(a.q) + (r.first + i) * a.q_token_stride +
                          (h * a.group + row - i * a.group) * a.q_head_stride;
#pragma unroll
            for (int i2 = 0; i2 < NQ; ++i2) {
                // 16-bit: piece i covers dims 32 i + 8 c ..; int8: 16 dims 64 (i / 2) + 16 c + 8 (i % 2)
                const int d = I8 ? 64 * (i2 >> 1) + 16 * c + 8 * (i2 & 1) : 32 * i2 + 8 * c;
                qf[n][i2] = live ? __ldg(reinterpret_cast<const uint4*>(qp + d)) : make_uint4(0, 0, 0, 0);
            }
            q_scale[n][0] = q_scale[n][1] = a.scale_log2;
            if constexpr (!std::is_same<C, T>::value) {
                // bf16 rows as fp16 times a power of two that brings the row's largest element to [2^14, 2^15): exact
                // for elements down to 2^-28 of the largest (smaller ones lose less than 2^-39 of it), so also where
                // the largest meets codes of 0.  Rows all below 2^-100 are lifted as those.
                float x[NQ][8], top = 0.0f;
#pragma unroll
                for (int i2 = 0; i2 < NQ; ++i2) {
                    load8(reinterpret_cast<const T*>(&qf[n][i2]), x[i2]);
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[i2][e]));
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127;
                ex = ex > 127 ? 0 : max(ex, -100) - 14;
                const float down = __int_as_float((127 - ex) << 23), up = __int_as_float((127 + ex) << 23);
#pragma unroll
                for (int i2 = 0; i2 < NQ; ++i2)
                    qf[n][i2] = make_uint4(pack2<C>(x[i2][0] * down, x[i2][1] * down), pack2<C>(x[i2][2] * down, x[i2][3] * down),
                                           pack2<C>(x[i2][4] * down, x[i2][5] * down), pack2<C>(x[i2][6] * down, x[i2][7] * down));
#pragma unroll
                for (int e = 0; e < 2; ++e)  // not 0, whose product with a masked score would be NaN
                    q_scale[n][e] = fmaxf(q_scale[n][e] * __shfl_sync(0xffffffffu, up, (2 * c + e) * 4), 1.17549435e-38f);
            }
        }
        // accumulator element 2 k + e of every tile: row 2 c + e (+ 8 n), key (or dim) g of half k
        int pos[NR][2];
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = 2 * c + e + 8 * n;
                pos[n][e] = row < rows ? r.len - r.n + row / a.group : -1;
            }

        float o[NR][NB][4][4];  // [.][block][w][2 k + e]: dim 64 block + 8 g + 2 w + k
        float m[NR][2], l[NR][2];  // m: the running maximum less kLift
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.0f;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int w = 0; w < 4; ++w)
#pragma unroll
                    for (int k = 0; k < 4; ++k) o[n][i][w][k] = 0.0f;
        }
        // int8: the weights times the V scales could leave fp16's range, so o[.][i] is kept in units of the
        // largest power of two not above any V scale of block i so far
        float unit[NB], inv_unit[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) unit[i] = inv_unit[i] = 0.0f;

        for (int it = it0; it < it1; ++it) {
            cp_async_wait<G::kStages - 1>();
            __syncwarp();
            const uint32_t st = ring + slot * G::kStage;
            // ---- scores: keys g and g + 8 of the 16 ----
            float s[NR][4];
            if constexpr (!I8) {
#pragma unroll
                for (int n = 0; n < NR; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) s[n][k] = 0.0f;
#pragma unroll
                for (int i = 0; i < NK; ++i) {
                    const uint4 x = lds128(st + k_read[i & 1] + (i >> 1) * 2048), y = lds128(st + k_read[i & 1] + (i >> 1) * 2048 + G::kEight);
#pragma unroll
                    for (int n = 0; n < NR; ++n) {
                        mma16816<C>(s[n], x.x, y.x, x.y, y.y, qf[n][i].x, qf[n][i].y);
                        mma16816<C>(s[n], x.z, y.z, x.w, y.w, qf[n][i].z, qf[n][i].w);
                    }
                }
            } else {
                // the codes are exact in 16 bits; a block's scale multiplies its fp32 dot product
                float blk[NR][NB][4];
#pragma unroll
                for (int i = 0; i < NB; ++i) {
#pragma unroll
                    for (int n = 0; n < NR; ++n)
#pragma unroll
                        for (int k = 0; k < 4; ++k) blk[n][i][k] = 0.0f;
                    const uint4 x = lds128(st + k_read[i & 1] + (i >> 1) * 2048), y = lds128(st + k_read[i & 1] + (i >> 1) * 2048 + G::kEight);
                    const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t x0, x1, y0, y1;
                        codes_to_pairs(xw[w], x0, x1);
                        codes_to_pairs(yw[w], y0, y1);
#pragma unroll
                        for (int n = 0; n < NR; ++n) {
                            const uint4 q = qf[n][2 * i + (w >> 1)];
                            mma16816<C>(blk[n][i], x0, y0, x1, y1, w & 1 ? q.z : q.x, w & 1 ? q.w : q.y);
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t sc = st + 2 * G::kKv + (8 * k + g) * 4 * NB;
                    float ks[NB];
#pragma unroll
                    for (int i = 0; i < NB; ++i) ks[i] = ldsf(sc + 4 * i);
#pragma unroll
                    for (int n = 0; n < NR; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float x = blk[n][0][2 * k + e] * ks[0];
                            if constexpr (NB == 2) x = fmaf(blk[n][1][2 * k + e], ks[1], x);
                            s[n][2 * k + e] = x;
                        }
                }
            }
            // ---- mask ----
            const uint32_t here = lds32(haves + slot * 4);
            if (here != 0xffffu || !same) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const bool in = here >> (8 * k + g) & 1u;
                    const int j = span.key(it * G::kTile + warp * 16 + 8 * k + g);
#pragma unroll
                    for (int n = 0; n < NR; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (!in || !(same || row_sees(a, pos[n][e], j))) s[n][2 * k + e] = -INFINITY;
                }
            }
            // ---- running maximum and sum; weights ----
            float p[NR][4];
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                float mx[2], al[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) mx[e] = fmaxf(s[n][e], s[n][2 + e]);
#pragma unroll
                for (int sh = 4; sh < 32; sh <<= 1)
#pragma unroll
                    for (int e = 0; e < 2; ++e) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], sh));
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float mn = fmaxf(m[n][e], fmaf(mx[e], q_scale[n][e], -kLift));
                    const float base = mn == -INFINITY ? 0.0f : mn;
                    al[e] = ex2(m[n][e] - base);
                    m[n][e] = mn;
                    p[n][e] = ex2(fmaf(s[n][e], q_scale[n][e], -base));
                    p[n][2 + e] = ex2(fmaf(s[n][2 + e], q_scale[n][e], -base));
                    l[n][e] = fmaf(l[n][e], al[e], p[n][e] + p[n][2 + e]);
                }
                if (__any_sync(0xffffffffu, al[0] != 1.0f || al[1] != 1.0f)) {
#pragma unroll
                    for (int i = 0; i < NB; ++i)
#pragma unroll
                        for (int w = 0; w < 4; ++w)
#pragma unroll
                            for (int k = 0; k < 4; ++k) o[n][i][w][k] *= al[k & 1];
                }
            }
            // ---- output ----
            uint32_t pb[NR][2];  // 16-bit: the weights as operands, the same for every block
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                uint32_t b0[NR], b1[NR];
                if constexpr (I8) {
                    float v0 = ldsf(st + 2 * G::kKv + (16 + g) * 4 * NB + 4 * i), v1 = ldsf(st + 2 * G::kKv + (24 + g) * 4 * NB + 4 * i);
                    if (__any_sync(0xffffffffu, fmaxf(v0, v1) >= 2.0f * unit[i])) {
                        float vm = fmaxf(v0, v1);
#pragma unroll
                        for (int sh = 4; sh < 32; sh <<= 1) vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, sh));
                        vm = __uint_as_float(__float_as_uint(vm) & 0x7f800000u);
                        if (vm > unit[i]) {
                            const float f = unit[i] * (1.0f / vm);
#pragma unroll
                            for (int n = 0; n < NR; ++n)
#pragma unroll
                                for (int w = 0; w < 4; ++w)
#pragma unroll
                                    for (int k = 0; k < 4; ++k) o[n][i][w][k] *= f;
                            unit[i] = vm;
                            inv_unit[i] = 1.0f / vm;
                        }
                    }
                    v0 *= inv_unit[i];
                    v1 *= inv_unit[i];
#pragma unroll
                    for (int n = 0; n < NR; ++n) {
                        b0[n] = transpose8(pack2<C>(p[n][0] * v0, p[n][1] * v0));
                        b1[n] = transpose8(pack2<C>(p[n][2] * v1, p[n][3] * v1));
                    }
                } else if (i == 0) {
#pragma unroll
                    for (int n = 0; n < NR; ++n) {
                        b0[n] = transpose8(pack2<C>(p[n][0], p[n][1]));
                        b1[n] = transpose8(pack2<C>(p[n][2], p[n][3]));
                        pb[n][0] = b0[n];
                        pb[n][1] = b1[n];
                    }
                } else {
#pragma unroll
                    for (int n = 0; n < NR; ++n) {
                        b0[n] = pb[n][0];
                        b1[n] = pb[n][1];
                    }
                }
                const uint32_t va = st + (I8 ? v_read[i][0] : v_read[0][0] + i * 2048), vb = st + (I8 ? v_read[i][1] : v_read[0][1] + i * 2048);
                if constexpr (I8) {
                    const uint2 f0 = lds64(va), f1 = lds64(vb), f2 = lds64(va + G::kEight), f3 = lds64(vb + G::kEight);
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t x0 = w >> 1 ? f0.y : f0.x, x1 = w >> 1 ? f1.y : f1.x, x2 = w >> 1 ? f2.y : f2.x, x3 = w >> 1 ? f3.y : f3.x;
                        const uint32_t sel = w & 1 ? 0x7362 : 0x5140;
                        uint32_t a0, a1, a2, a3;
                        codes_to_pairs(__byte_perm(x0, x1, sel), a0, a1);
                        codes_to_pairs(__byte_perm(x2, x3, sel), a2, a3);
#pragma unroll
                        for (int n = 0; n < NR; ++n) mma16816<C>(o[n][i][w], a0, a1, a2, a3, b0[n], b1[n]);
                    }
                } else {
                    const uint4 f0 = lds128(va), f1 = lds128(vb), f2 = lds128(va + G::kEight), f3 = lds128(vb + G::kEight);
                    const uint32_t w0[4] = {f0.x, f0.y, f0.z, f0.w}, w1[4] = {f1.x, f1.y, f1.z, f1.w};
                    const uint32_t w2[4] = {f2.x, f2.y, f2.z, f2.w}, w3[4] = {f3.x, f3.y, f3.z, f3.w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t a0 = __byte_perm(w0[w], w1[w], 0x5410), a1 = __byte_perm(w0[w], w1[w], 0x7632);
                        const uint32_t a2 = __byte_perm(w2[w], w3[w], 0x5410), a3 = __byte_perm(w2[w], w3[w], 0x7632);
#pragma unroll
                        for (int n = 0; n < NR; ++n) mma16816<C>(o[n][i][w], a0, a1, a2, a3, b0[n], b1[n]);
                    }
                }
            }
            __syncwarp();
            const int nx = it + G::kStages;
            if (nx < it1) {
                const int odd = (nx - it0) & 1;
                if (!odd) {
                    prepare(nx, pg);
                    pg = lookup(nx + 2);
                }
                issue(slot, odd);
            }
            cp_async_commit();
            slot = slot + 1 == G::kStages ? 0 : slot + 1;
        }
        cp_async_wait<0>();
        if constexpr (I8) {
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int i = 0; i < NB; ++i)
#pragma unroll
                    for (int w = 0; w < 4; ++w)
#pragma unroll
                        for (int k = 0; k < 4; ++k) o[n][i][w][k] *= unit[i];
        }
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int sh = 4; sh < 32; sh <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], sh);
        // ---- join the warps: the ring's memory holds their (max, sum, output) ----
        __syncthreads();
        float* mo = reinterpret_cast<float*>(rows_smem);
        float* mm = mo + G::kWarps * 16 * G::kMergeRow;
        float* ml = mm + G::kWarps * 16;
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = warp * 16 + 2 * c + e + 8 * n;
                if (2 * c + e + 8 * n >= rows) continue;
                if (g == 0) {
                    mm[row] = m[n][e];
                    ml[row] = l[n][e];
                }
#pragma unroll
                for (int i = 0; i < NB; ++i)
#pragma unroll
                    for (int w = 0; w < 4; w += 2)
                        *reinterpret_cast<float4*>(mo + row * G::kMergeRow + 64 * i + 8 * g + 2 * w) =
                            make_float4(o[n][i][w][e], o[n][i][w][2 + e], o[n][i][w + 1][e], o[n][i][w + 1][2 + e]);
            }
        __syncthreads();
        // a row of the joined result: DP dims per thread, from n results of it `stride` rows apart
        constexpr int DP = 8, kPer = D / DP;
        const bool split = c0 > 0 || c1 < chunks;
        constexpr int PF = part_floats(16, D);
        float* mine = a.part + static_cast<long long>(2 * blockIdx.x + (x == begin ? 0 : 1)) * PF;
        auto store = [&](int row, int d0, float(&acc)[DP], float mx, float sum) {
            const int i = row / a.group;
            const long long qh = static_cast<long long>(r.first + i) * a.heads + h * a.group + (row - i * a.group);
            attention_store<T, DP>(a, 0, qh, D, d0, d0 == 0, acc, mx, sum);
        };
        for (int row = tid / kPer; row < rows; row += G::kThreads / kPer) {
            const int d0 = tid % kPer * DP;
            float acc[DP], mx = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < G::kWarps; ++w) mx = fmaxf(mx, mm[w * 16 + row]);
            const float base = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
            for (int d = 0; d < DP; ++d) acc[d] = 0.0f;
#pragma unroll
            for (int w = 0; w < G::kWarps; ++w) {
                const float f = ex2(mm[w * 16 + row] - base);
                sum = fmaf(ml[w * 16 + row], f, sum);
#pragma unroll
                for (int d = 0; d < DP; ++d) acc[d] = fmaf(mo[(w * 16 + row) * G::kMergeRow + d0 + d], f, acc[d]);
            }
            if (split) {
#pragma unroll
                for (int d = 0; d < DP; d += 4)
                    *reinterpret_cast<float4*>(mine + row * D + d0 + d) = make_float4(acc[d], acc[d + 1], acc[d + 2], acc[d + 3]);
                if (tid % kPer == 0) *reinterpret_cast<float2*>(mine + 16 * D + 2 * row) = make_float2(mx, sum);
            } else {
                store(row, d0, acc, mx, sum);
            }
        }
        // ---- a unit split over CTAs: the last to arrive merges the parts in CTA order ----
        if (split) {
            const int ca = cta_of(unit_x), n = cta_of(unit_x + chunks - 1) - ca + 1;
            __threadfence();
            __syncthreads();
            if (tid == 0) s_last = atomicInc(a.count + static_cast<long long>(req) * kv_heads + h, n - 1) == static_cast<unsigned>(n - 1);
            __syncthreads();
            if (s_last) {
                __threadfence();
                const float* first = a.part + static_cast<long long>(2 * ca + (start_of(ca) == unit_x ? 0 : 1)) * PF;
                const float* rest = a.part + static_cast<long long>(2 * ca) * PF;  // part i > 0: slot 0 of CTA ca + i
                auto part = [&](int i) { return i == 0 ? first : rest + static_cast<long long>(2 * i) * PF; };
                // a row's warps: all maxima and sums first, then their share of the outputs, many loads at once
                const int subs = rows < G::kWarps ? G::kWarps / rows : 1;  // warps per row
                constexpr int kRowLanes = D / 4, kSide = 32 / kRowLanes;   // lanes of a row, parts side by side
                constexpr int kBatch = 8;
                const int d0 = lane % kRowLanes * 4, side = lane / kRowLanes;
                for (int t = warp; t < rows * subs; t += G::kWarps) {
                    const int row = t % rows, sub = t / rows;
                    float top = -INFINITY, sum = 0.0f;
                    for (int i = lane; i < n; i += 32) top = fmaxf(top, __ldcg(part(i) + 16 * D + 2 * row));
                    top = warp_max(top);
                    const float base = top == -INFINITY ? 0.0f : top;
                    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int i0p = sub * kSide + side; i0p < n; i0p += kBatch * subs * kSide) {
                        float4 v[kBatch];
                        float2 w[kBatch];
#pragma unroll
                        for (int k = 0; k < kBatch; ++k) {
                            const int i = i0p + k * subs * kSide;
                            v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            w[k] = make_float2(-INFINITY, 0.0f);
                            if (i < n) {
                                const float* pp = part(i);
                                v[k] = __ldcg(reinterpret_cast<const float4*>(pp + row * D + d0));
                                w[k] = __ldcg(reinterpret_cast<const float2*>(pp + 16 * D + 2 * row));
                            }
                        }
#pragma unroll
                        for (int k = 0; k < kBatch; ++k) {
                            const float f = ex2(w[k].x - base);
                            sum = fmaf(w[k].y, f, sum);
                            acc.x = fmaf(v[k].x, f, acc.x);
                            acc.y = fmaf(v[k].y, f, acc.y);
                            acc.z = fmaf(v[k].z, f, acc.z);
                            acc.w = fmaf(v[k].w, f, acc.w);
                        }
                    }
                    if constexpr (kSide == 2) {
                        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                        acc.x += __shfl_xor_sync(0xffffffffu, acc.x, 16);
                        acc.y += __shfl_xor_sync(0xffffffffu, acc.y, 16);
                        acc.z += __shfl_xor_sync(0xffffffffu, acc.z, 16);
                        acc.w += __shfl_xor_sync(0xffffffffu, acc.w, 16);
                    }
                    if (side == 0) *reinterpret_cast<float4*>(mo + (sub * 16 + row) * G::kMergeRow + d0) = acc;
                    if (lane == 0) {
                        mm[sub * 16 + row] = top;
                        ml[sub * 16 + row] = sum;
                    }
                }
                __syncthreads();
                for (int row = tid / kPer; row < rows; row += G::kThreads / kPer) {
                    const int d0 = tid % kPer * DP;
                    float acc[DP], sum = 0.0f;
#pragma unroll
                    for (int d = 0; d < DP; ++d) acc[d] = 0.0f;
                    for (int w = 0; w < subs; ++w) {
                        sum += ml[w * 16 + row];
#pragma unroll
                        for (int d = 0; d < DP; ++d) acc[d] += mo[(w * 16 + row) * G::kMergeRow + d0 + d];
                    }
                    store(row, d0, acc, mm[row], sum);
                }
            }
        }
        x = unit_x + c1;
        __syncthreads();  // the ring's memory is free again
    }
}

}  // namespace asdsl
