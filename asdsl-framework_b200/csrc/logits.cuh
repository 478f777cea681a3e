// logits.cuh -- penalties for repeated tokens, biases and grammar masks on a batch's logits.
#pragma once

#include "paged_cache.cuh"

namespace asdsl {

struct LogitsArgs {
    const void* in;             // [n][vocab], row stride in_stride
    void* out;                  // [n][vocab], row stride out_stride (may be `in`)
    long long in_stride, out_stride;
    const int32_t* tokens;      // [n][tokens_len] prompt then output ids, row stride tokens_stride (or null)
    long long tokens_stride;
    int tokens_len;
    const int32_t* lens;        // [n] ids in use
    const int32_t* prompt_lens; // [n] of them the prompt's
    const float* repetition;    // [n] or null
    const float* frequency;
    const float* presence;
    const int32_t* bias_ptr;    // [n + 1] or null
    const int32_t* bias_ids;
    const float* bias_values;
    int n_bias;
    const int32_t* mask;        // [n][mask_words], row stride mask_stride; bit v % 32 of word v / 32, 0 = forbidden
    long long mask_stride;
    int n, vocab;
};

constexpr int kLogitsThreads = 512;
constexpr int kLogitsList = kLogitsThreads;  // bias entries of a row kept in shared memory
constexpr int kLogitsVecs = 4;           // 16-byte accesses of a thread in a chunk of the stream
constexpr int kTouchSlots = 16384;       // ids of one round of k_logits_touch
constexpr int kTouchProbes = 64;
constexpr int kTouchWarps = kLogitsThreads / 32, kTouchList = kTouchSlots / kTouchWarps;  // ids that a warp lists
constexpr uint32_t kNoId = 0xffffffffu;
constexpr uint32_t kSeenBit = 0x80000000u, kBiasBit = 0x40000000u, kCountMask = 0x3fffffffu;

template <typename T>
__device__ __forceinline__ float load1(const T* p) {
    if constexpr (std::is_same<T, __half>::value) return __half2float(*p);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat162float(*p);
    else return *p;
}
template <typename T>
__device__ __forceinline__ void store1(T* p, float x) {
    if constexpr (std::is_same<T, __half>::value) *p = __float2half_rn(x);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) *p = __float2bfloat16_rn(x);
    else *p = x;
}

__device__ __forceinline__ bool allowed(const int32_t* mask, int v) {
    return !mask || (static_cast<uint32_t>(mask[v >> 5]) >> (v & 31) & 1u);
}

// The logits as they are, a forbidden id -inf whatever its logit held: one pass bound by memory.  Two CTAs
// per SM walk the (row, chunk) pairs, so that k_logits_touch, its programmatic dependent, runs beside them.
// (One kernel for both took 62 to 137 us for 128 rows of 200064 bf16 logits with 8000-id histories: every
// chunk's CTA worked through the whole history or waited, chunk by chunk, for its touched ids' values.)
template <typename T>
__global__ void __launch_bounds__(kLogitsThreads, 3) k_logits_stream(const LogitsArgs a) {
    constexpr int V = 16 / sizeof(T), kChunk = kLogitsThreads * kLogitsVecs * V;
    grid_launch_dependents();
    const int chunks = (a.vocab + kChunk - 1) / kChunk;
    const long long items = static_cast<long long>(a.n) * chunks;
    for (long long it = blockIdx.x; it < items; it += gridDim.x) {
        const int b = static_cast<int>(it / chunks), chunk = static_cast<int>(it - static_cast<long long>(b) * chunks);
        const T* in = static_cast<const T*>(a.in) + b * a.in_stride;
        T* out = static_cast<T*>(a.out) + b * a.out_stride;
        const int32_t* mask = a.mask ? a.mask + b * a.mask_stride : nullptr;
        // ids before the row's first 16-byte boundary belong to chunk 0; rows of `in` and `out` that do not
        // share it are walked one id at a time
        const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(in) & 15u) / sizeof(T));
        const bool vec = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
        const int pre = mis ? V - mis : 0;
        const int v0 = chunk == 0 ? 0 : min(a.vocab, pre + chunk * kChunk), v1 = min(a.vocab, pre + (chunk + 1) * kChunk);
        auto one = [&](int v) {
            if (allowed(mask, v)) out[v] = in[v];
            else store1(out + v, -INFINITY);
        };
        if (!vec) {
            for (int v = v0 + threadIdx.x; v < v1; v += kLogitsThreads) one(v);
            continue;
        }
        const int body = chunk == 0 ? min(pre, v1) : v0;  // first id on a 16-byte boundary
        const int n_vec = (v1 - body) / V;
        uint4 x[kLogitsVecs];
        uint32_t bits[kLogitsVecs];
#pragma unroll
        for (int i = 0; i < kLogitsVecs; ++i) {
            const int k = i * kLogitsThreads + threadIdx.x, v = body + k * V;
            bits[i] = 0xffffffffu;
            if (k < n_vec) {
                x[i] = __ldcs(reinterpret_cast<const uint4*>(in + v));
                if (mask) {
                    const int w = v >> 5, s = v & 31;
                    bits[i] = static_cast<uint32_t>(mask[w]) >> s;
                    if (s + V > 32) bits[i] |= static_cast<uint32_t>(mask[w + 1]) << (32 - s);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kLogitsVecs; ++i) {
            const int k = i * kLogitsThreads + threadIdx.x, v = body + k * V;
            if (k >= n_vec) break;
            uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
            constexpr uint32_t kLow = std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;  // -inf of a 16-bit type
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (V == 4) {
                    if (!(bits[i] >> e & 1u)) w[e] = 0xff800000u;
                } else {
                    if (!(bits[i] >> (2 * e) & 1u)) w[e] = (w[e] & 0xffff0000u) | kLow;
                    if (!(bits[i] >> (2 * e + 1) & 1u)) w[e] = (w[e] & 0xffffu) | kLow << 16;
                }
            }
            *reinterpret_cast<uint4*>(out + v) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        // the ids before the first and after the last 16-byte access
        if (static_cast<int>(threadIdx.x) < body - v0) one(v0 + threadIdx.x);
        const int tail = body + n_vec * V;
        if (static_cast<int>(threadIdx.x) < v1 - tail) one(tail + threadIdx.x);
    }
}

// a value in place of its counts: its inverted bits, never 0
__device__ __forceinline__ uint32_t touched_word(float y) { return y != y ? ~0x7fc00000u : ~__float_as_uint(y); }

// The ids that a request's history or bias list touches: counted in a hash table in shared memory (a
// request has few thousand, whatever the vocabulary), their values computed from the logits, and written
// over the stream's.  Integer additions give the same counts in any order; an id's bias entries are added
// in list order.
//
// One CTA per request; with gridDim.x > 1, for histories too long for one, CTA p of them takes the ids
// p * kTouchSlots .. of the vocabulary, each its own slot.  A table that overflows (more distinct ids than
// the probes find room for) is given up for rounds over such ranges.
template <typename T>
__global__ void __launch_bounds__(kLogitsThreads, 3) k_logits_touch(const LogitsArgs a) {
    extern __shared__ __align__(16) uint32_t touch_smem[];
    uint32_t* key = touch_smem;                 // [kTouchSlots]
    uint32_t* word = touch_smem + kTouchSlots;  // [kTouchSlots] counts and bits, then the value
    unsigned short* listed = reinterpret_cast<unsigned short*>(touch_smem + 2 * kTouchSlots);  // [kTouchWarps][kTouchList]
    __shared__ int s_ids[kLogitsThreads];
    __shared__ float s_values[kLogitsThreads];
    __shared__ int s_full, s_twice;
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    listed += (tid >> 5) * kTouchList;
    const T* in = static_cast<const T*>(a.in) + b * a.in_stride;
    T* out = static_cast<T*>(a.out) + b * a.out_stride;
    const int32_t* mask = a.mask ? a.mask + b * a.mask_stride : nullptr;
    const int len = a.tokens ? min(max(a.lens[b], 0), a.tokens_len) : 0;
    const int prompt = a.tokens && a.prompt_lens ? a.prompt_lens[b] : 0;
    const float rep = a.repetition ? a.repetition[b] : 1.0f, freq = a.frequency ? a.frequency[b] : 0.0f,
                pres = a.presence ? a.presence[b] : 0.0f;
    int e0 = 0, e1 = 0;
    if (a.bias_ptr) {
        e0 = min(max(a.bias_ptr[b], 0), a.n_bias);
        e1 = max(min(a.bias_ptr[b + 1], a.n_bias), e0);
    }
    const int32_t* tk = a.tokens + b * a.tokens_stride;
    if (e0 + tid < e1) {  // the list's first entries; later ones are read where they are
        s_ids[tid] = a.bias_ids[e0 + tid];
        s_values[tid] = a.bias_values[e0 + tid];
    }
    bool hashed = gridDim.x == 1 && a.vocab > kTouchSlots, waited = false;
    int v0 = hashed ? 0 : blockIdx.x * kTouchSlots;
    while (v0 < a.vocab) {
        const int v1 = hashed ? a.vocab : min(a.vocab, v0 + kTouchSlots);
        for (int i = tid; i < kTouchSlots / 4; i += kLogitsThreads) {
            reinterpret_cast<uint4*>(word)[i] = make_uint4(0, 0, 0, 0);
            if (hashed) reinterpret_cast<uint4*>(key)[i] = make_uint4(kNoId, kNoId, kNoId, kNoId);
        }
        if (tid == 0) s_full = s_twice = 0;
        __syncthreads();
        // the slot of an id (-1: none free), and whether it was free before
        auto slot_of = [&](int id, bool& fresh) {
            if (!hashed) return id - v0;
            uint32_t s = (static_cast<uint32_t>(id) * 2654435761u) >> 18;
            static_assert(kTouchSlots == 1 << 14, "14 bits of the product");
            for (int probe = 0; probe < kTouchProbes; ++probe, s = (s + 1) & (kTouchSlots - 1)) {
                uint32_t k = *static_cast<volatile uint32_t*>(key + s);
                if (k == kNoId) {
                    k = atomicCAS(key + s, kNoId, static_cast<uint32_t>(id));
                    fresh = k == kNoId;
                }
                if (k == kNoId || k == static_cast<uint32_t>(id)) return static_cast<int>(s);
            }
            s_full = 1;
            return -1;
        };
        int n_listed = 0;  // of this warp
        auto list = [&](bool fresh, int s) {
            __syncwarp();
            const unsigned m = __ballot_sync(0xffffffffu, fresh);
            const int at = n_listed + __popc(m & ((1u << lane) - 1));
            if (fresh && at < kTouchList) listed[at] = static_cast<unsigned short>(s);
            n_listed += __popc(m);
        };
        constexpr int kUnroll = 8;
        for (int i0 = tid - lane; i0 < len; i0 += kUnroll * kLogitsThreads) {
            int id[kUnroll];
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                const int i = i0 + lane + k * kLogitsThreads;
                id[k] = i < len ? tk[i] : -1;
            }
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                bool fresh = false;
                int s = -1;
                if (id[k] >= v0 && id[k] < v1) {
                    s = slot_of(id[k], fresh);
                    if (s >= 0) {
                        if (i0 + lane + k * kLogitsThreads >= prompt) atomicAdd(word + s, 1u);
                        else if (!(*static_cast<volatile uint32_t*>(word + s) & kSeenBit)) atomicOr(word + s, kSeenBit);
                    }
                }
                list(fresh, s);
            }
        }
        for (int i0 = tid - lane; i0 < e1 - e0; i0 += kLogitsThreads) {
            const int i = i0 + lane, id = i >= e1 - e0 ? -1 : (i < kLogitsThreads ? s_ids[i] : a.bias_ids[e0 + i]);
            bool fresh = false;
            int s = -1;
            if (id >= v0 && id < v1) {
                s = slot_of(id, fresh);
                if (s >= 0 && (atomicOr(word + s, kBiasBit) & kBiasBit)) s_twice = 1;
            }
            list(fresh, s);
        }
        if (n_listed > kTouchList) s_full = 1;
        __syncthreads();
        if (s_full) {
            hashed = false;
            __syncthreads();
            continue;
        }
        // x = seen ? (x > 0 ? x / r : x * r) : x;  x -= f * count + p * [count > 0];  the loads of a few slots
        // at once
        constexpr int kSlots = 8;
        const int j_first = hashed ? lane : tid, j_step = hashed ? 32 : kLogitsThreads, j_end = hashed ? n_listed : kTouchSlots;
        auto slot_at = [&](int j) { return hashed ? listed[min(j, kTouchList - 1)] : j & (kTouchSlots - 1); };
        for (int j0 = j_first; j0 < j_end; j0 += kSlots * j_step) {
            uint32_t cnt[kSlots];
            T x[kSlots];
#pragma unroll
            for (int k = 0; k < kSlots; ++k) {
                const int j = j0 + k * j_step, s = j < j_end ? slot_at(j) : 0;
                cnt[k] = j < j_end ? word[s] : 0u;
                // without a branch, so that the loads go out together: an untouched slot loads the first logit
                x[k] = in[cnt[k] ? (hashed ? static_cast<int>(key[s]) : v0 + s) : 0];
            }
#pragma unroll
            for (int k = 0; k < kSlots; ++k) {
                if (!cnt[k]) continue;
                float y = load1(&x[k]);
                if (cnt[k] & ~kBiasBit) {
                    y = y > 0.0f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
                    const uint32_t c = cnt[k] & kCountMask;
                    if (c) y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, static_cast<float>(c))), pres);
                }
                word[slot_at(j0 + k * j_step)] = touched_word(y);
            }
        }
        __syncthreads();
        // x += biases: where no id is listed twice every entry by itself, else by the id's first entry, whose
        // warp adds the later ones in list order
        if (!s_twice) {
            for (int i = tid; i < e1 - e0; i += kLogitsThreads) {
                const int id = i < kLogitsThreads ? s_ids[i] : a.bias_ids[e0 + i];
                if (id < v0 || id >= v1) continue;
                const float x = i < kLogitsThreads ? s_values[i] : a.bias_values[e0 + i];
                bool fresh;
                uint32_t* w = word + slot_of(id, fresh);
                if (x != 0.0f) *w = touched_word(__uint_as_float(~*w) + x);
            }
        } else {
            for (int i = tid >> 5; i < e1 - e0; i += kLogitsThreads / 32) {
                const int id = i < kLogitsThreads ? s_ids[i] : a.bias_ids[e0 + i];
                if (id < v0 || id >= v1) continue;
                float sum = 0.0f;
                bool later = false;
                for (int k0 = 0; k0 < e1 - e0 && !later; k0 += 32) {
                    const int k = k0 + lane;
                    const bool hit = k < e1 - e0 && (k < kLogitsThreads ? s_ids[k] : a.bias_ids[e0 + k]) == id;
                    for (unsigned h = __ballot_sync(0xffffffffu, hit); h; h &= h - 1) {
                        const int at = k0 + __ffs(h) - 1;
                        later = later || at < i;
                        sum += at < kLogitsThreads ? s_values[at] : a.bias_values[e0 + at];
                    }
                }
                if (!later && lane == 0 && sum != 0.0f) {
                    bool fresh;
                    uint32_t* w = word + slot_of(id, fresh);
                    *w = touched_word(__uint_as_float(~*w) + sum);
                }
            }
        }
        __syncthreads();
        if (!waited) grid_dependency_wait();
        waited = true;
        for (int j0 = j_first; j0 < j_end; j0 += kSlots * j_step) {
            uint32_t w[kSlots], bits[kSlots];
            int v[kSlots];
#pragma unroll
            for (int k = 0; k < kSlots; ++k) {
                const int j = j0 + k * j_step, s = j < j_end ? slot_at(j) : 0;
                w[k] = j < j_end ? word[s] : 0u;
                v[k] = w[k] ? (hashed ? static_cast<int>(key[s]) : v0 + s) : 0;
                bits[k] = mask ? static_cast<uint32_t>(mask[v[k] >> 5]) : 0xffffffffu;
            }
#pragma unroll
            for (int k = 0; k < kSlots; ++k)  // a forbidden id stays as the stream wrote it
                if (w[k] && (bits[k] >> (v[k] & 31) & 1u)) store1(out + v[k], __uint_as_float(~w[k]));
        }
        if (hashed || gridDim.x > 1) break;
        v0 += kTouchSlots;
        __syncthreads();
    }
    if (!waited) grid_dependency_wait();
}

// Both in one launch, for batches of few chunks: one CTA per (16 bytes of each thread, request).  Its logits
// and mask words are loaded first, so that their latency passes while the touched ids' values are worked
// out in shared memory from the whole history; the stream is then a select per logit.
template <typename T>
__global__ void __launch_bounds__(kLogitsThreads) k_logits_few(const LogitsArgs a) {
    constexpr int V = 16 / sizeof(T), kIds = kLogitsThreads * V;
    // of id v at v - body + V: 0 untouched; counts; then the inverted bits of its value
    __shared__ __align__(16) uint32_t logits_word[kIds + 2 * V];
    __shared__ uint32_t s_biased[(kIds + 2 * V + 31) / 32];
    __shared__ int s_ids[kLogitsList];
    __shared__ float s_values[kLogitsList];
    __shared__ int s_twice;
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    const T* in = static_cast<const T*>(a.in) + b * a.in_stride;
    T* out = static_cast<T*>(a.out) + b * a.out_stride;
    // rows of `in` and `out` that do not share their 16-byte boundary are walked one id at a time
    const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(in) & 15u) / sizeof(T));
    const int pre = mis ? V - mis : 0;
    const bool vec = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
    const int v0 = blockIdx.x == 0 ? 0 : pre + blockIdx.x * kIds;
    const int v1 = min(a.vocab, pre + static_cast<int>(blockIdx.x + 1) * kIds);
    if (v1 <= v0) return;
    const int body = blockIdx.x == 0 ? min(pre, v1) : v0;  // first id on a 16-byte boundary
    const int n_vec = vec ? (v1 - body) / V : 0;
    const int32_t* mask = a.mask ? a.mask + b * a.mask_stride : nullptr;
    const int vb = body + tid * V;  // this thread's access
    uint4 x = make_uint4(0, 0, 0, 0);
    uint32_t bits = 0xffffffffu;
    if (tid < n_vec) {
        x = *reinterpret_cast<const uint4*>(in + vb);
        if (mask) {
            const int w = vb >> 5, s = vb & 31;
            bits = static_cast<uint32_t>(mask[w]) >> s;
            if (s + V > 32) bits |= static_cast<uint32_t>(mask[w + 1]) << (32 - s);
        }
    }
    const int len = a.tokens ? min(max(a.lens[b], 0), a.tokens_len) : 0;
    const int prompt = a.tokens && a.prompt_lens ? a.prompt_lens[b] : 0;
    const float rep = a.repetition ? a.repetition[b] : 1.0f, freq = a.frequency ? a.frequency[b] : 0.0f,
                pres = a.presence ? a.presence[b] : 0.0f;
    int e0 = 0, e1 = 0;
    if (a.bias_ptr) {
        e0 = min(max(a.bias_ptr[b], 0), a.n_bias);
        e1 = max(min(a.bias_ptr[b + 1], a.n_bias), e0);
    }
    if (e0 + tid < e1) {  // the list's first entries; later ones are read where they are
        s_ids[tid] = a.bias_ids[e0 + tid];
        s_values[tid] = a.bias_values[e0 + tid];
    }
    for (int i = tid; i < (kIds + 2 * V) / 4; i += kLogitsThreads) reinterpret_cast<uint4*>(logits_word)[i] = make_uint4(0, 0, 0, 0);
    for (int i = tid; i < (kIds + 2 * V + 31) / 32; i += kLogitsThreads) s_biased[i] = 0;
    if (tid == 0) s_twice = 0;
    const int base = body - V;  // id of logits_word[0]
    __syncthreads();
    // x = seen ? (x > 0 ? x / r : x * r) : x;  x -= f * count + p * [count > 0]
    auto penalised = [&](int v, uint32_t cnt) {
        float y = load1(in + v);
        y = y > 0.0f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
        const uint32_t c = cnt & kCountMask;
        if (c) y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, static_cast<float>(c))), pres);
        return touched_word(y);
    };
    if (len > 0) {
        const int32_t* tk = a.tokens + b * a.tokens_stride;
        constexpr int kUnroll = 8;
        for (int i0 = tid; i0 < len; i0 += kUnroll * kLogitsThreads) {
            int id[kUnroll];
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                const int i = i0 + k * kLogitsThreads;
                id[k] = i < len ? tk[i] : -1;
            }
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                if (id[k] < v0 || id[k] >= v1) continue;
                uint32_t* w = logits_word + (id[k] - base);
                if (i0 + k * kLogitsThreads >= prompt) atomicAdd(w, 1u);
                else atomicOr(w, kSeenBit);
            }
        }
        __syncthreads();
#pragma unroll 1
        for (int v = v0 + tid; v < v1; v += kLogitsThreads) {
            const uint32_t cnt = logits_word[v - base];
            if (cnt) logits_word[v - base] = penalised(v, cnt);
        }
    }
    if (e1 > e0) {
        for (int i = tid; i < e1 - e0; i += kLogitsThreads) {
            const int id = i < kLogitsList ? s_ids[i] : a.bias_ids[e0 + i];
            if (id < v0 || id >= v1) continue;
            const uint32_t bit = 1u << ((id - base) & 31);
            if (atomicOr(s_biased + ((id - base) >> 5), bit) & bit) s_twice = 1;
        }
        __syncthreads();
        // where no id is listed twice every entry adds itself, else the id's first entry, whose warp adds the
        // later ones in list order
        auto add = [&](int id, float y) {
            uint32_t* w = logits_word + (id - base);
            if (y != 0.0f) *w = touched_word((*w ? __uint_as_float(~*w) : load1(in + id)) + y);
        };
        if (!s_twice) {
            for (int i = tid; i < e1 - e0; i += kLogitsThreads) {
                const int id = i < kLogitsList ? s_ids[i] : a.bias_ids[e0 + i];
                if (id >= v0 && id < v1) add(id, i < kLogitsList ? s_values[i] : a.bias_values[e0 + i]);
            }
        } else {
            for (int i = tid >> 5; i < e1 - e0; i += kLogitsThreads / 32) {
                const int id = i < kLogitsList ? s_ids[i] : a.bias_ids[e0 + i];
                if (id < v0 || id >= v1) continue;
                float sum = 0.0f;
                bool later = false;
                for (int k0 = 0; k0 < e1 - e0 && !later; k0 += 32) {
                    const int k = k0 + lane;
                    const bool hit = k < e1 - e0 && (k < kLogitsList ? s_ids[k] : a.bias_ids[e0 + k]) == id;
                    for (unsigned h = __ballot_sync(0xffffffffu, hit); h; h &= h - 1) {
                        const int at = k0 + __ffs(h) - 1;
                        later = later || at < i;
                        sum += at < kLogitsList ? s_values[at] : a.bias_values[e0 + at];
                    }
                }
                if (!later && lane == 0) add(id, sum);
            }
        }
    }
    __syncthreads();
    auto one = [&](int v) {
        const uint32_t w = logits_word[v - base];
        const bool may = !mask || (static_cast<uint32_t>(mask[v >> 5]) >> (v & 31) & 1u);
        if (!may) store1(out + v, -INFINITY);
        else if (w) store1(out + v, __uint_as_float(~w));
        else out[v] = in[v];
    };
    if (!vec) {
        for (int v = v0 + tid; v < v1; v += kLogitsThreads) one(v);
        return;
    }
    if (tid < n_vec) {
        uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < V; e += 4) {
            const uint4 t = *reinterpret_cast<const uint4*>(logits_word + V + tid * V + e);
            const uint32_t tw[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool may = bits >> (e + j) & 1u;
                if constexpr (V == 4) {
                    if (tw[j]) w[j] = ~tw[j];
                    if (!may) w[j] = 0xff800000u;
                } else {
                    const float y = may ? __uint_as_float(~tw[j]) : -INFINITY;
                    if (tw[j] || !may) {
                        const uint32_t h = pack2<T>(y, y);
                        const int q = (e + j) >> 1;
                        w[q] = (j & 1) ? __byte_perm(w[q], h, 0x5410) : __byte_perm(w[q], h, 0x3254);
                    }
                }
            }
        }
        *reinterpret_cast<uint4*>(out + vb) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    // the ids before the first and after the last 16-byte access
    if (tid < body - v0) one(v0 + tid);
    const int tail = body + n_vec * V;
    if (tid < v1 - tail) one(tail + tid);
}

}  // namespace asdsl
