// batch_api.cuh -- the C entry points that serve a batch over a paged cache (include/asdsl_b200.h).
// Included by asdsl_b200.cu.
#pragma once

#include <algorithm>
#include <atomic>
#include <cmath>

#include "attention_tiles.cuh"
#include "launch.cuh"
#include "logits.cuh"

namespace asdsl {

// Shared memory above 48 KB is opted into once per kernel and device.
template <auto Kern>
inline int allow_smem(int bytes) {
    static std::atomic<unsigned long long> done{0};  // one bit per device
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return kOk;
    ASDSL_CUDA(cudaFuncSetAttribute(reinterpret_cast<const void*>(Kern), cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_relaxed);
    return kOk;
}

// launch as a programmatic dependent of the kernel before it on the stream (which calls
// grid_launch_dependents) or, with pdl false, as an ordinary kernel
template <typename A>
inline int launch_dependent(void (*kern)(A), dim3 grid, int threads, int smem, bool pdl, cudaStream_t st, const A& args) {
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    ASDSL_CUDA(cudaLaunchKernelEx(&cfg, kern, args));
    return kOk;
}

// An SM's split between L1 and shared memory changes only when it is idle: a kernel that is to run beside
// one that needs shared memory asks for all of it.
template <auto Kern>
inline int prefer_smem() {
    static std::atomic<unsigned long long> done{0};  // one bit per device
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return kOk;
    ASDSL_CUDA(cudaFuncSetAttribute(reinterpret_cast<const void*>(Kern), cudaFuncAttributePreferredSharedMemoryCarveout,
                                    cudaSharedmemCarveoutMaxShared));
    done.fetch_or(bit, std::memory_order_relaxed);
    return kOk;
}

inline bool batch_dtype(int t) { return t == ASDSL_B200_F32 || t == ASDSL_B200_BF16 || t == ASDSL_B200_F16; }

inline int check_cache(const asdsl_b200_paged_cache* c, const char* fn, CacheView* out) {
    const std::string f(fn);
    if (!c || !c->k || !c->v) return set_error(kEinval, f + ": null cache");
    if (c->dtype != ASDSL_B200_BF16 && c->dtype != ASDSL_B200_F16 && c->dtype != ASDSL_B200_I8)
        return set_error(kEinval, f + ": the cache must be bf16, fp16 or int8");
    if (c->head_dim != 64 && c->head_dim != 128) return set_error(kEinval, f + ": head_dim must be 64 or 128");
    if (c->n_pages <= 0 || c->page_size <= 0 || c->kv_heads <= 0) return set_error(kEinval, f + ": invalid cache dimensions");
    if (static_cast<long long>(c->n_pages) * c->page_size > 0x7fffffffll)
        return set_error(kEinval, f + ": the cache holds more than 2^31 - 1 positions");
    const bool i8 = c->dtype == ASDSL_B200_I8;
    if (i8 && (!c->k_scales || !c->v_scales)) return set_error(kEinval, f + ": an int8 cache needs scales");
    if (!aligned16(c->k) || !aligned16(c->v) || (i8 && (!aligned16(c->k_scales) || !aligned16(c->v_scales))))
        return set_error(kEinval, f + ": cache buffers must be 16-byte aligned");
    const long long unit = i8 ? 16 : 8;
    if (c->page_stride % unit || c->token_stride % unit || c->head_stride % unit || c->page_stride < 0 ||
        c->token_stride < 0 || c->head_stride < 0)
        return set_error(kEinval, f + ": cache strides must be multiples of 16 bytes");
    out->k = c->k;
    out->v = c->v;
    out->ks = c->k_scales;
    out->vs = c->v_scales;
    out->page_stride = c->page_stride;
    out->token_stride = c->token_stride;
    out->head_stride = c->head_stride;
    out->n_pages = c->n_pages;
    out->kv_heads = c->kv_heads;
    out->page = FastDiv::make(c->page_size);
    return kOk;
}

// ---- attention dispatch --------------------------------------------------------------------
// Workspace: partial results of split units of the few-rows kernel, parts of split rows of the
// many-rows kernel (both fixed areas per device), then the arrival counters.
inline size_t attention_part_bytes() {
    return static_cast<size_t>(2 * kRowsMaxCtas) * sm_count() * part_floats(16, 128) * sizeof(float);
}
inline long long attention_part_rows() { return static_cast<long long>(kUnitRows) * sm_count(); }
inline size_t attention_rows_bytes() { return static_cast<size_t>(attention_part_rows()) * (128 + 2) * sizeof(float); }

template <typename T, bool I8, int D, int NR>
inline int launch_rows(const AttnPagedArgs& a, cudaStream_t st) {
    constexpr int smem = RowsGeom<I8, D>::kSmem;
    if (int rc = allow_smem<k_attention_rows_paged<T, I8, D, NR>>(smem)) return rc;
    k_attention_rows_paged<T, I8, D, NR><<<RowsGeom<I8, D>::kCtas * sm_count(), RowsGeom<I8, D>::kThreads, smem, st>>>(a);
    ASDSL_CUDA(cudaGetLastError());
    return kOk;
}

template <typename T, bool I8, int D>
inline int launch_tiles(const AttnPagedArgs& a, long long grid, cudaStream_t st) {
    using G = TileGeom<I8, D>;
    static std::atomic<unsigned long long> checked{0};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!(checked.load(std::memory_order_relaxed) >> (dev & 63) & 1u)) {
        // the warpgroups' register split must fit what the block is launched with, or it would wait forever
        cudaFuncAttributes at;
        ASDSL_CUDA(cudaFuncGetAttributes(&at, k_attention_tiles_paged<T, I8, D>));
        if (at.numRegs * kTileThreads < 256 * (kSoftmaxRegs + kOtherRegs))
            return set_error(kEcuda, "attention: kernel built with too few registers");
        checked.fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
    }
    if (int rc = allow_smem<k_attention_tiles_paged<T, I8, D>>(G::kSmem)) return rc;
    if (grid > 0x7fffffffll) return set_error(kEinval, "attention: too many rows");
    k_attention_tiles_paged<T, I8, D><<<static_cast<unsigned>(grid), kTileThreads, G::kSmem, st>>>(a);
    ASDSL_CUDA(cudaGetLastError());
    return kOk;
}

constexpr int kMinTilesPerSplit = 4;
constexpr int kManyKeys = 2048;  // from here 9 to 16 rows of a single request go to the many-rows kernel

// What a launch left in parts: where their maxima and sums lie (behind the outputs), and how many there are.
struct AttnParts {
    float2* ml;
    int n;
};

// All rows joined from their parts.
template <typename T, int D>
inline int launch_join(AttnPagedArgs a, cudaStream_t st) {
    constexpr int per = 256 / (D / 8);
    const long long rows = static_cast<long long>(a.tokens) * a.heads;
    k_attention_join<T, D><<<static_cast<unsigned>((rows + per - 1) / per), 256, 0, st>>>(a);
    ASDSL_CUDA(cudaGetLastError());
    return kOk;
}

// Which kernel takes which requests.  Up to 16 rows (tokens x group heads of a KV head) are one
// tensor-core tile of the few-rows kernel, bound by the cache's bytes; more go to the many-rows
// kernel: 64 requests of 16 rows on 4000 bf16 / int8 keys (8 KV heads of 128) take 209 / 270 us in the
// few-rows kernel and 260 / 463 us in the other, 8 requests 59 / 68 and 53 / 76 us.  The host knows
// lengths only where every request has one row or there is one request; in a batch of ragged rows both
// kernels run and each passes over the other's requests.
template <typename T, bool I8, int D>
inline int launch_attention_as(AttnPagedArgs a, float* rows_ws, AttnParts* parts, cudaStream_t st) {
    const long long rows = static_cast<long long>(a.tokens) * a.heads;
    const long long all_rows = static_cast<long long>(a.tokens) * a.group;
    const bool one_each = a.lens && !a.cu, single = !a.lens || a.n_req == 1;
    long long keys = a.lens ? static_cast<long long>(a.width) * a.c.page.d : a.const_len;
    if (a.causal && a.window > 0) keys = std::min(keys, static_cast<long long>(a.sinks) + a.window + kUnitRows / a.group + 1);
    // One request alone is split over all SMs by either kernel, and joining 9 to 16 rows costs the few-rows kernel
    // more than a part-filled tile costs the other: 16 rows of 8 KV heads on 1000 / 2000 / 8000 / 64000 bf16 keys
    // 20 / 27 / 51 / 94 us, many-rows 22 / 22 / 29 / 76 us; int8 22 / 29 / 53 / 111 and 25 / 25 / 33 / 115 us.  `keys`
    // is what the table can hold: with fewer keys in it the loss is the 2 us of the short lengths.
    const long long few_rows = single && keys >= kManyKeys && !one_each ? kSmallRows / 2 : kSmallRows;
    const bool only_few = one_each ? a.group <= kSmallRows : all_rows <= few_rows;
    const bool only_many = !only_few && (one_each || single);
    a.small_rows = only_many ? 0 : kSmallRows;
    if (!only_few) {
        // an upper bound of the 256-row blocks, and key splits while those leave SMs idle
        const long long reqs = only_many ? a.n_req : std::min<long long>(a.n_req, all_rows / (kSmallRows + 1));
        const long long blocks = one_each ? static_cast<long long>(a.n_req) * ((a.group + kUnitRows - 1) / kUnitRows)
                                          : (!a.lens || a.n_req == 1 ? (all_rows + kUnitRows - 1) / kUnitRows
                                                                     : all_rows / kUnitRows + reqs);
        const long long ctas = blocks * a.c.kv_heads;
        const long long iters = (keys + TileGeom<I8, D>::kKeys - 1) / TileGeom<I8, D>::kKeys;
        long long splits = ctas > 0 ? sm_count() / ctas : 1;
        splits = std::min(splits, iters / kMinTilesPerSplit);
        if (a.parts_ml || splits < 1) splits = 1;  // (the part of a joined call is one)
        a.splits = static_cast<int>(splits);
        a.splits_last = 0;
        long long grid = ctas * splits;
        // One request whose last block is a single row tile: its CTAs take about half the time per key, so it gets
        // half the parts and the other blocks the SMs that this frees.
        const long long last_rows = all_rows % kUnitRows;
        if (splits > 1 && blocks > 1 && (!a.lens || a.n_req == 1) && last_rows > 0 && last_rows <= kTileRows) {
            const long long per_head = sm_count() / a.c.kv_heads;
            long long s = per_head / (blocks - 1);
            while (s > 1 && s * (blocks - 1) + (s + 1) / 2 > per_head) --s;
            s = std::min(s, iters / kMinTilesPerSplit);
            if (s > splits) {
                splits = s;
                a.splits = static_cast<int>(s);
                a.splits_last = static_cast<int>((s + 1) / 2);
                grid = (s * (blocks - 1) + a.splits_last) * a.c.kv_heads;
            }
        }
        const bool join = splits > 1 && !a.parts_acc;
        AttnPagedArgs k = a;
        if (join) k.parts_acc = rows_ws;
        // a prefix leaves room for one more part
        if (k.parts_acc && !k.parts_ml) k.parts_ml = reinterpret_cast<float2*>(k.parts_acc + (splits + (join ? 0 : 1)) * rows * D);
        if (parts) *parts = AttnParts{k.parts_ml, a.splits};
        if (int rc = launch_tiles<T, I8, D>(k, grid, st)) return rc;
        if (join) {
            k.n_parts = a.splits;
            if (int rc = launch_join<T, D>(k, st)) return rc;
        }
    }
    if (only_many) return kOk;
    if (a.parts_acc && !a.parts_ml) {
        a.parts_ml = reinterpret_cast<float2*>(a.parts_acc + 2 * rows * D);
        if (parts) *parts = AttnParts{a.parts_ml, 1};
    }
    // one row tile of 8 where every request has at most 8 rows, else two
    const bool eight = one_each ? a.group <= 8 : all_rows <= 8;
    return eight ? launch_rows<T, I8, D, 1>(a, st) : launch_rows<T, I8, D, 2>(a, st);
}

// A call with parts_acc set leaves parts instead of rows: of all rows as one request (a prefix), where
// `parts` says how many and where, or with parts_ml set one part of each row.
inline int launch_attention(const AttnPagedArgs& a, int q_dtype, int cache_dtype, int D, float* rows_ws, AttnParts* parts,
                            cudaStream_t st) {
    const bool i8 = cache_dtype == ASDSL_B200_I8, half = q_dtype == ASDSL_B200_F16;
    if (D == 64) {
        if (half) return i8 ? launch_attention_as<__half, true, 64>(a, rows_ws, parts, st) : launch_attention_as<__half, false, 64>(a, rows_ws, parts, st);
        return i8 ? launch_attention_as<__nv_bfloat16, true, 64>(a, rows_ws, parts, st) : launch_attention_as<__nv_bfloat16, false, 64>(a, rows_ws, parts, st);
    }
    if (half) return i8 ? launch_attention_as<__half, true, 128>(a, rows_ws, parts, st) : launch_attention_as<__half, false, 128>(a, rows_ws, parts, st);
    return i8 ? launch_attention_as<__nv_bfloat16, true, 128>(a, rows_ws, parts, st) : launch_attention_as<__nv_bfloat16, false, 128>(a, rows_ws, parts, st);
}

template <typename T>
inline int launch_logits(const LogitsArgs& a, cudaStream_t st) {
    constexpr int V = 16 / static_cast<int>(sizeof(T)), narrow = kLogitsThreads * V, wide = narrow * kLogitsVecs;
    // One launch while the chunks are few (each reads its row's whole history): one row of 200064 fp32 logits
    // and 500 ids 6.3 us, against 8.9 us of the two kernels; 128 rows of bf16 with 8000 ids 105 us against 49.
    const long long few = static_cast<long long>(a.n) * ((a.vocab + narrow - 1) / narrow);
    if (few <= 4 * sm_count()) {
        k_logits_few<T><<<dim3((a.vocab + narrow - 1) / narrow, a.n), kLogitsThreads, 0, st>>>(a);
        ASDSL_CUDA(cudaGetLastError());
        return kOk;
    }
    const bool touch = a.tokens || a.bias_ptr;
    // in place without a mask the stream would change nothing
    const bool stream = a.mask || a.in != a.out || a.in_stride != a.out_stride;
    if (stream) {
        if (int rc = prefer_smem<k_logits_stream<T>>()) return rc;
        const long long items = static_cast<long long>(a.n) * ((a.vocab + wide - 1) / wide);
        k_logits_stream<T><<<static_cast<unsigned>(std::min<long long>(items, 2 * sm_count())), kLogitsThreads, 0, st>>>(a);
        ASDSL_CUDA(cudaGetLastError());
    }
    if (!touch) return kOk;
    constexpr int smem = kTouchSlots * (4 + 4 + 2);
    if (int rc = allow_smem<k_logits_touch<T>>(smem)) return rc;
    // a history that may hold more distinct ids than the table takes is split by ranges of ids
    const unsigned parts = a.tokens_len > kTouchSlots / 2 + kTouchSlots / 4 ? (a.vocab + kTouchSlots - 1) / kTouchSlots : 1;
    return launch_dependent(k_logits_touch<T>, dim3(parts, a.n), kLogitsThreads, smem, stream, st, a);
}

inline int attention_args(const char* fn, AttnPagedArgs* a, const void* q, int q_dtype, long long q_token_stride,
                          long long q_head_stride, const asdsl_b200_paged_cache* cache, const int32_t* table,
                          long long table_stride, int width, const int32_t* lens, const int32_t* cu, int n_req, int tokens,
                          int heads, float scale, void* out, float* lse, void* ws, size_t ws_bytes) {
    const std::string f(fn);
    std::memset(a, 0, sizeof(*a));
    if (int rc = check_cache(cache, fn, &a->c)) return rc;
    if (q_dtype != ASDSL_B200_BF16 && q_dtype != ASDSL_B200_F16) return set_error(kEinval, f + ": q must be bf16 or fp16");
    if (cache->dtype != ASDSL_B200_I8 && cache->dtype != q_dtype)
        return set_error(kEinval, f + ": a 16-bit cache must have the type of q");
    if (n_req < 0 || tokens < 0 || heads <= 0 || heads % cache->kv_heads || width < 0)
        return set_error(kEinval, f + ": invalid dimensions (heads must be a multiple of kv_heads)");
    if (!(scale > 0.0f) || std::isinf(scale)) return set_error(kEinval, f + ": scale must be positive and finite");
    if (static_cast<long long>(tokens) * heads > 0x7fffffffll) return set_error(kEinval, f + ": too many rows");
    if (!cu && n_req != tokens) return set_error(kEinval, f + ": without row starts every request has one row");
    if (tokens > 0 && n_req > 0 && (!q || !out || !lens || (width > 0 && !table) || !ws)) return set_error(kEinval, f + ": null pointer");
    if (!aligned16(q) || !aligned16(out) || q_token_stride % 8 || q_head_stride % 8)
        return set_error(kEinval, f + ": q and out must be 16-byte aligned with strides of multiples of 16 bytes");
    if (!aligned16(ws) || (tokens > 0 && n_req > 0 && ws_bytes < asdsl_b200_attention_workspace_bytes(n_req, tokens, heads, cache->kv_heads)))
        return set_error(kEinval, f + ": workspace too small or not 16-byte aligned");
    a->q = q;
    a->q_token_stride = q_token_stride;
    a->q_head_stride = q_head_stride;
    a->table = table;
    a->table_stride = table_stride;
    a->width = width;
    a->lens = lens;
    a->cu = cu;
    a->n_req = n_req;
    a->tokens = tokens;
    a->heads = heads;
    a->group = heads / cache->kv_heads;
    a->by_group = FastDiv::make(a->group);
    a->causal = 1;
    a->scale_log2 = scale * 1.44269504088896341f;
    a->out = out;
    a->lse = lse;
    a->part = static_cast<float*>(ws);
    a->count = reinterpret_cast<unsigned int*>(static_cast<char*>(ws) + attention_part_bytes() + attention_rows_bytes());
    return kOk;
}

}  // namespace asdsl

using namespace asdsl;

extern "C" {

int asdsl_b200_plan_step(const int32_t* kv_lens, const int32_t* new_lens, int n_requests, const int32_t* free_pages,
                         int n_free, int page_size, int32_t* block_table, long long table_stride, int table_width,
                         int32_t* cu_q, int32_t* total_lens, int32_t* slots, int32_t* positions, int32_t* requests,
                         int max_tokens, int32_t* counts, void* stream) {
    if (n_requests < 0 || n_requests > kPlanMaxRequests)
        return set_error(kEinval, "plan_step: 0 to " + std::to_string(kPlanMaxRequests) + " requests");
    if (n_free < 0 || page_size <= 0 || table_width < 0 || max_tokens < 0 || table_stride < table_width)
        return set_error(kEinval, "plan_step: invalid dimensions");
    if (!cu_q || !counts || (n_requests > 0 && (!kv_lens || !new_lens || !total_lens)) ||
        (n_requests > 0 && table_width > 0 && !block_table) || (n_free > 0 && !free_pages) ||
        (max_tokens > 0 && (!slots || !positions || !requests)))
        return set_error(kEinval, "plan_step: null pointer");
    // every CTA reads the inputs for as long as it runs, whatever the others have written
    const auto shared = [&](const void* out, long long out_n) {
        const auto meets = [&](const void* in, long long in_n) {
            const uintptr_t x = reinterpret_cast<uintptr_t>(in), y = reinterpret_cast<uintptr_t>(out);
            return in_n > 0 && out_n > 0 && x < y + static_cast<uintptr_t>(out_n) * 4 && y < x + static_cast<uintptr_t>(in_n) * 4;
        };
        return meets(kv_lens, n_requests) || meets(new_lens, n_requests) || meets(free_pages, n_free);
    };
    if (shared(block_table, n_requests > 0 && table_width > 0 ? (n_requests - 1) * table_stride + table_width : 0) ||
        shared(cu_q, n_requests + 1) || shared(total_lens, n_requests) || shared(slots, max_tokens) ||
        shared(positions, max_tokens) || shared(requests, max_tokens) || shared(counts, 3))
        return set_error(kEinval, "plan_step: the lengths and free_pages must not overlap what the step writes");
    PlanArgs a;
    a.kv_lens = kv_lens;
    a.new_lens = new_lens;
    a.free_pages = free_pages;
    a.table = block_table;
    a.cu = cu_q;
    a.total = total_lens;
    a.slots = slots;
    a.positions = positions;
    a.requests = requests;
    a.counts = counts;
    a.table_stride = table_stride;
    a.n = n_requests;
    a.n_free = n_free;
    a.width = table_width;
    a.max_tokens = max_tokens;
    a.page = FastDiv::make(page_size);
    const int smem = 2 * (n_requests + 1) * static_cast<int>(sizeof(int32_t));
    if (int rc = allow_smem<k_plan_step>(2 * (kPlanMaxRequests + 1) * static_cast<int>(sizeof(int32_t)))) return rc;
    // one token per thread up to two CTAs per SM; a decode step's few tokens are one CTA
    const long long want = (static_cast<long long>(max_tokens) + kPlanThreads - 1) / kPlanThreads;
    const int grid = static_cast<int>(want < 1 ? 1 : (want > 2 * sm_count() ? 2 * sm_count() : want));
    k_plan_step<<<grid, kPlanThreads, smem, static_cast<cudaStream_t>(stream)>>>(a);
    ASDSL_CUDA(cudaGetLastError());
    return kOk;
}

int asdsl_b200_kv_write(const asdsl_b200_paged_cache* cache, const void* k, const void* v, int dtype,
                        long long token_stride, long long head_stride, const int32_t* slots, int n_tokens, void* stream) {
    KvWriteArgs a;
    if (int rc = check_cache(cache, "kv_write", &a.c)) return rc;
    if (!batch_dtype(dtype)) return set_error(kEinval, "kv_write: k and v must be fp32, bf16 or fp16");
    if (cache->dtype != ASDSL_B200_I8 && dtype != ASDSL_B200_F32 && dtype != cache->dtype)
        return set_error(kEinval, "kv_write: a 16-bit cache takes its own type or fp32");
    if (n_tokens < 0) return set_error(kEinval, "kv_write: invalid dimensions");
    if (n_tokens == 0) return kOk;
    if (!k || !v || !slots) return set_error(kEinval, "kv_write: null pointer");
    const int unit = dtype == ASDSL_B200_F32 ? 4 : 8;
    if (!aligned16(k) || !aligned16(v) || token_stride % unit || head_stride % unit)
        return set_error(kEinval, "kv_write: k and v must be 16-byte aligned with strides of multiples of 16 bytes");
    a.k = k;
    a.v = v;
    a.token_stride = token_stride;
    a.head_stride = head_stride;
    a.slots = slots;
    a.tokens = n_tokens;
    a.head_dim = cache->head_dim;
    if (static_cast<long long>(n_tokens) * cache->kv_heads > 0x7fffffffll) return set_error(kEinval, "kv_write: too many rows");
    a.heads = FastDiv::make(cache->kv_heads);
    a.items = static_cast<long long>(n_tokens) * cache->kv_heads * (cache->head_dim / 8);
    const unsigned grid = static_cast<unsigned>((a.items + 255) / 256);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (cache->dtype == ASDSL_B200_I8) {
        if (dtype == ASDSL_B200_F32) k_kv_write<float, int8_t><<<grid, 256, 0, st>>>(a);
        else if (dtype == ASDSL_B200_BF16) k_kv_write<__nv_bfloat16, int8_t><<<grid, 256, 0, st>>>(a);
        else k_kv_write<__half, int8_t><<<grid, 256, 0, st>>>(a);
    } else if (cache->dtype == ASDSL_B200_BF16) {
        if (dtype == ASDSL_B200_F32) k_kv_write<float, __nv_bfloat16><<<grid, 256, 0, st>>>(a);
        else k_kv_write<__nv_bfloat16, __nv_bfloat16><<<grid, 256, 0, st>>>(a);
    } else {
        if (dtype == ASDSL_B200_F32) k_kv_write<float, __half><<<grid, 256, 0, st>>>(a);
        else k_kv_write<__half, __half><<<grid, 256, 0, st>>>(a);
    }
    ASDSL_CUDA(cudaGetLastError());
    return kOk;
}

size_t asdsl_b200_attention_workspace_bytes(int n_requests, int n_tokens, int heads, int kv_heads) {
    if (n_requests < 0 || n_tokens < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads) return 0;
    return attention_part_bytes() + attention_rows_bytes() + static_cast<size_t>(n_requests) * kv_heads * sizeof(unsigned int);
}

size_t asdsl_b200_attention_merge_bytes(int n_tokens, int heads, int head_dim) {
    if (n_tokens < 0 || heads <= 0 || head_dim <= 0) return 0;
    return static_cast<size_t>(std::max(static_cast<long long>(n_tokens) * heads, attention_part_rows()) + static_cast<long long>(n_tokens) * heads) * (head_dim + 2) * sizeof(float);
}

int asdsl_b200_attention_paged(const void* q, int q_dtype, long long q_token_stride, long long q_head_stride,
                               const asdsl_b200_paged_cache* cache, const int32_t* block_table, long long table_stride,
                               int table_width, const int32_t* kv_lens, const int32_t* cu_q, int n_requests, int n_tokens,
                               int heads, int window, int sinks, float scale, void* out, float* lse, void* workspace,
                               size_t workspace_bytes, void* stream) {
    AttnPagedArgs a;
    if (window < 0 || sinks < 0) return set_error(kEinval, "attention_paged: window and sinks must not be negative");
    if (int rc = attention_args("attention_paged", &a, q, q_dtype, q_token_stride, q_head_stride, cache, block_table,
                                table_stride, table_width, kv_lens, cu_q, n_requests, n_tokens, heads, scale, out, lse,
                                workspace, workspace_bytes))
        return rc;
    if (n_tokens == 0 || n_requests == 0) return kOk;
    a.window = window;
    a.sinks = sinks;
    float* rows_ws = reinterpret_cast<float*>(static_cast<char*>(workspace) + attention_part_bytes());
    return launch_attention(a, q_dtype, cache->dtype, cache->head_dim, rows_ws, nullptr, static_cast<cudaStream_t>(stream));
}

int asdsl_b200_attention_shared_prefix(const void* q, int q_dtype, long long q_token_stride, long long q_head_stride,
                                       const asdsl_b200_paged_cache* cache, const int32_t* prefix_pages, int n_prefix_pages,
                                       int prefix_len, const int32_t* block_table, long long table_stride, int table_width,
                                       const int32_t* kv_lens, const int32_t* cu_q, int n_requests, int n_tokens, int heads,
                                       float scale, void* out, float* lse, void* merge_scratch, size_t merge_bytes,
                                       void* workspace, size_t workspace_bytes, void* stream) {
    AttnPagedArgs a;
    if (int rc = attention_args("attention_shared_prefix", &a, q, q_dtype, q_token_stride, q_head_stride, cache, block_table,
                                table_stride, table_width, kv_lens, cu_q, n_requests, n_tokens, heads, scale, out, lse,
                                workspace, workspace_bytes))
        return rc;
    if (prefix_len < 0 || n_prefix_pages < 0 ||
        prefix_len > static_cast<long long>(n_prefix_pages) * cache->page_size)
        return set_error(kEinval, "attention_shared_prefix: prefix_len must lie within the prefix's pages");
    if (n_tokens == 0 || n_requests == 0) return kOk;
    if ((prefix_len > 0 && !prefix_pages) || !merge_scratch || !aligned16(merge_scratch))
        return set_error(kEinval, "attention_shared_prefix: null or misaligned pointer");
    if (merge_bytes < asdsl_b200_attention_merge_bytes(n_tokens, heads, cache->head_dim))
        return set_error(kEinval, "attention_shared_prefix: merge scratch too small");
    float* merge = static_cast<float*>(merge_scratch);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    float* rows_ws = reinterpret_cast<float*>(static_cast<char*>(workspace) + attention_part_bytes());
    if (prefix_len > 0) {
        AttnPagedArgs p = a;  // all rows as one request over the prefix
        p.table = prefix_pages;
        p.table_stride = n_prefix_pages;
        p.width = n_prefix_pages;
        p.lens = nullptr;
        p.const_len = prefix_len;
        p.cu = nullptr;
        p.n_req = 1;
        p.causal = 0;
        p.parts_acc = merge;
        AttnParts parts{nullptr, 0};
        if (int rc = launch_attention(p, q_dtype, cache->dtype, cache->head_dim, rows_ws, &parts, st)) return rc;
        const long long rows = static_cast<long long>(n_tokens) * heads;
        AttnPagedArgs own = a;
        own.parts_acc = merge + parts.n * rows * cache->head_dim;
        own.parts_ml = parts.ml + parts.n * rows;
        if (int rc = launch_attention(own, q_dtype, cache->dtype, cache->head_dim, rows_ws, nullptr, st)) return rc;
        a.parts_acc = merge;
        a.parts_ml = parts.ml;
        a.n_parts = parts.n + 1;
        const bool half = q_dtype == ASDSL_B200_F16;
        if (cache->head_dim == 64) return half ? launch_join<__half, 64>(a, st) : launch_join<__nv_bfloat16, 64>(a, st);
        return half ? launch_join<__half, 128>(a, st) : launch_join<__nv_bfloat16, 128>(a, st);
    }
    return launch_attention(a, q_dtype, cache->dtype, cache->head_dim, rows_ws, nullptr, st);
}

int asdsl_b200_logits_process(const void* logits, void* out, int dtype, long long in_stride, long long out_stride, int n,
                              int vocab, const int32_t* tokens, long long tokens_stride, int tokens_len, const int32_t* lens,
                              const int32_t* prompt_lens, const float* repetition, const float* frequency,
                              const float* presence, const int32_t* bias_ptr, const int32_t* bias_ids,
                              const float* bias_values, int n_bias, const int32_t* mask, long long mask_stride, void* stream) {
    if (!batch_dtype(dtype)) return set_error(kEinval, "logits_process: logits must be fp32, bf16 or fp16");
    if (n < 0 || vocab <= 0 || tokens_len < 0 || n_bias < 0 || n > 65535 || vocab > (1 << 30))
        return set_error(kEinval, "logits_process: invalid dimensions");
    if (n == 0) return kOk;
    if (!logits || !out || (tokens && !lens) || (bias_ptr && n_bias > 0 && (!bias_ids || !bias_values)))
        return set_error(kEinval, "logits_process: null pointer");
    const int es = dtype == ASDSL_B200_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(logits) % es || reinterpret_cast<uintptr_t>(out) % es)
        return set_error(kEinval, "logits_process: misaligned logits");
    LogitsArgs a;
    std::memset(&a, 0, sizeof(a));
    a.in = logits;
    a.out = out;
    a.in_stride = in_stride;
    a.out_stride = out_stride;
    a.tokens = tokens_len > 0 ? tokens : nullptr;
    a.tokens_stride = tokens_stride;
    a.tokens_len = tokens_len;
    a.lens = lens;
    a.prompt_lens = prompt_lens;
    a.repetition = repetition;
    a.frequency = frequency;
    a.presence = presence;
    a.bias_ptr = n_bias > 0 ? bias_ptr : nullptr;
    a.bias_ids = bias_ids;
    a.bias_values = bias_values;
    a.n_bias = n_bias;
    a.mask = mask;
    a.mask_stride = mask_stride;
    a.n = n;
    a.vocab = vocab;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int rc = kOk;
    if (dtype == ASDSL_B200_F32) rc = launch_logits<float>(a, st);
    else if (dtype == ASDSL_B200_BF16) rc = launch_logits<__nv_bfloat16>(a, st);
    else rc = launch_logits<__half>(a, st);
    if (rc) return rc;
    ASDSL_CUDA(cudaGetLastError());
    return kOk;
}

}  // extern "C"
