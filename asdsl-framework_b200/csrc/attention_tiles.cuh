// attention_tiles.cuh -- attention of a batch over a paged cache: many query rows per request (prompts,
// drafts under verification, a batch's rows against a shared prefix) on the 5th-generation tensor cores.
//
// One CTA takes up to 256 query rows (tokens x group heads) of a request and KV head as two tiles of
// 128 rows (a TMEM lane per row) and walks their keys in tiles of 128 (64 for int8 pages):
//
//   loaders  (4 warps)   keys and values, gathered page by page, into 128-byte-swizzled shared memory
//   issuer   (1 thread)  S = Q K^T into TMEM, O += P V with P read from TMEM
//   softmax  (2 x 4 warps, one thread per row)  S from TMEM, running maximum and sum, P back to TMEM
//
// While one tile's softmax runs, the tensor cores work on the other tile.  P overwrites S in place, so
// the order of issue (O += P V before the next S of the same tile) is all the synchronisation that the
// reuse needs.  The running maximum moves only when it grows by more than 2^kSlack (the weights stay below
// that, exact in the sum and the same relative rounding in P), so the accumulator in TMEM is rescaled
// rarely (a known method): 2^8, for fp16 2^3, which leaves the weights more of its range (kLift, as in the
// few-rows kernel).  8192 fp16 rows on 16384 keys with 2^3 / 2^8: 1250 / 1247 us with scores of unit spread, 1320
// / 1260 us with three times that, where rows' maxima still grow late.
//
// int8 pages: the codes are exact in 16 bits; S of each 64-dim block is a separate accumulator that the
// softmax multiplies by the block's K scale in fp32, and P is multiplied by the V scale of each block
// before its one rounding.  For fp16 those products are kept in range by a power of two per block and row
// tile, as in the few-rows kernel.
#pragma once

#include "attention_paged.cuh"
#include "launch.cuh"

namespace asdsl {

// ---- tcgen05 -------------------------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t* smem_dst, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_dst)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t addr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// D (TMEM) = A (shared) B (shared) [+ D]
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(acc))
        : "memory");
}
// D (TMEM) = A (TMEM) B (shared) [+ D]
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(acc))
        : "memory");
}
// 32 consecutive 32-bit columns of this thread's TMEM lane
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
        "%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
// Ties the registers of an asynchronous TMEM load to this point: placed after the wait, it keeps their
// uses from being scheduled before it.
__device__ __forceinline__ void reg_fence32(uint32_t (&r)[32]) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]));
    asm volatile("" : "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,"
        "%31,%32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

// two fp32 operations in one instruction
__device__ __forceinline__ uint64_t pack_f32x2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Shared-memory operand descriptor, 128-byte swizzle (rows of 128 bytes, atoms of 8 rows, 1024-byte
// aligned): lbo / sbo in bytes.  K-major: sbo = 8 rows (lbo unused).  MN-major: sbo = 8 rows along K,
// lbo = the next 64 elements along N.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return static_cast<uint64_t>((addr >> 4) & 0x3fffu) | (static_cast<uint64_t>((lbo >> 4) & 0x3fffu) << 16) |
           (static_cast<uint64_t>((sbo >> 4) & 0x3fffu) << 32) | (1ull << 46) | (2ull << 61);
}
// kind::f16 instruction descriptor: fp32 accumulator, A K-major, M = 128
template <typename T>
__device__ __forceinline__ constexpr uint32_t tc_idesc(uint32_t n, bool b_mn_major) {
    constexpr uint32_t t = std::is_same<T, __half>::value ? 0u : 1u;
    return (1u << 4) | (t << 7) | (t << 10) | (static_cast<uint32_t>(b_mn_major) << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

template <typename T>
__device__ __forceinline__ void codes_to_pairs_as(uint32_t w, uint32_t& p01, uint32_t& p23) {
    if constexpr (std::is_same<T, __half>::value) {
        codes_to_pairs(w, p01, p23);
    } else {
        const uint32_t m = w & 0x7f7f7f7fu, s = w & 0x80808080u;
        uint32_t x0 = __byte_perm(m, 0x43434343u, 0x4140), x1 = __byte_perm(m, 0x43434343u, 0x4342);
        uint32_t y0 = __byte_perm(s, 0x43434343u, 0x4140), y1 = __byte_perm(s, 0x43434343u, 0x4342);
        const __nv_bfloat162 r0 = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&x0), *reinterpret_cast<__nv_bfloat162*>(&y0));
        const __nv_bfloat162 r1 = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&x1), *reinterpret_cast<__nv_bfloat162*>(&y1));
        p01 = *reinterpret_cast<const uint32_t*>(&r0);
        p23 = *reinterpret_cast<const uint32_t*>(&r1);
    }
}

// ---- geometry ------------------------------------------------------------------------------
constexpr int kTileThreads = 512;  // softmax A, softmax B, loaders, issuer (a warpgroup each)
// registers per thread of the softmax warpgroups and of the other two: the sum must not pass what the
// block is launched with (128 each)
constexpr int kSoftmaxRegs = 200, kOtherRegs = 56;
constexpr int kTileRows = 128;
constexpr int kUnitRows = 2 * kTileRows;
constexpr int kSmallRows = 16;     // requests with no more rows than this go to the few-rows kernel (the launch rule has the figures)
constexpr int kMetaSlots = 4;      // > key tiles between the loaders and the slower softmax

template <bool I8, int D>
struct TileGeom {
    static constexpr int kKeys = I8 ? 64 : 128;           // keys per tile
    static constexpr int kHalves = D / 64;                // 64-dim chunks of 128-byte rows
    static constexpr int kQ = kTileRows * D * 2;          // bytes of a Q tile
    static constexpr int kOp = kKeys * D * 2;             // bytes of a K or V tile as an operand
    static constexpr int kStages = 4;                     // K and V tiles in turn: two key tiles
    static constexpr int kRawCodes = kKeys * D * 2;       // int8: codes of a K and a V tile before conversion,
    static constexpr int kRaw = I8 ? kRawCodes + 128 * 16 : 0;  // then 16 bytes per loader thread: scales, presence
    static constexpr int kRawStages = I8 ? 4 : 0;
    static constexpr int kMeta = 16 + (I8 ? 2 * kKeys * kHalves * 4 : 0);  // which keys exist, scales
    static constexpr int kBytes = 2 * kQ + kStages * kOp + kRawStages * kRaw + kMetaSlots * kMeta;
    static constexpr int kSmem = kBytes + 1024;           // the base is rounded up to 1024
};

struct TileBars {
    uint64_t q_full, full[4], empty[4], meta[kMetaSlots], s_full[2], p_ready[2][2], o_done[2];
};

// Bounded wait that also gives up once another role has: `dead` is in shared memory.
__device__ __forceinline__ bool tile_wait(uint64_t* bar, uint32_t parity, volatile int* dead) {
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long t0 = globaltimer_ns();
    while (true) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*dead) return false;
        if (globaltimer_ns() - t0 > kWaitLimitNs) {
            *dead = 1;
            atomicOr(&g_status_word, static_cast<unsigned int>(kStatusWaitFull));
            return false;
        }
    }
}

template <typename T, bool I8, int D>
__global__ void __launch_bounds__(kTileThreads, 1) k_attention_tiles_paged(const AttnPagedArgs a) {
    using G = TileGeom<I8, D>;
    constexpr int BK = G::kKeys;
    constexpr int NH = G::kHalves;
    extern __shared__ uint8_t tile_smem_raw[];
    __shared__ TileBars bars;
    __shared__ uint32_t s_tmem;
    __shared__ int s_scan[kTileThreads / 32], s_req, s_blk;
    __shared__ volatile int s_dead;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    // ---- which unit: the block-th block of 256 rows, counted over the requests from the last ----
    // (with splits_last set, the first CTAs take the last block of the only request in fewer parts)
    int split, splits = a.splits, h, block;
    {
        int x = blockIdx.x;
        const int last = a.splits_last * a.c.kv_heads;
        if (x < last) {
            splits = a.splits_last;
            block = 0;
        } else {
            x -= last;
            block = x / (splits * a.c.kv_heads) + (last > 0 ? 1 : 0);
        }
        split = x % splits;
        h = x / splits % a.c.kv_heads;
    }
    auto blocks_of = [&](const ReqRows& r) {
        const int rows = r.n * a.group;
        return rows > a.small_rows ? (rows + kUnitRows - 1) / kUnitRows : 0;
    };
    if (tid == 0) {
        s_req = -1;
        s_dead = 0;
    }
    int total = 0;
    const bool once = a.n_req <= kTileThreads;  // else a second pass finds the request
    for (int pass = 0; pass < (once ? 1 : 2); ++pass) {
        int base = 0;
        for (int r0 = 0; r0 < a.n_req; r0 += kTileThreads) {
            const int cnt = r0 + tid < a.n_req ? blocks_of(request_rows(a, r0 + tid)) : 0;
            int inc = cnt;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += t;
            }
            if (lane == 31) s_scan[warp] = inc;
            __syncthreads();
            int before = base;
#pragma unroll
            for (int w = 0; w < kTileThreads / 32; ++w) {
                if (w < warp) before += s_scan[w];
                base += s_scan[w];
            }
            if (once) total = base;
            if (once || pass == 1) {
                const int want = total - 1 - block, mine = before + inc - cnt;
                if (want >= mine && want < mine + cnt) {
                    s_req = r0 + tid;
                    s_blk = want - mine;
                }
            }
            __syncthreads();
        }
        if (pass == 0) {
            total = base;
            if (block >= total) return;
        }
    }
    const int req = s_req;
    const ReqRows r = request_rows(a, req);
    const int row0 = s_blk * kUnitRows, rows = min(kUnitRows, r.n * a.group - row0);
    const bool two = rows > kTileRows;
    const KeySpan span = key_span(a, r, row0 / a.group, (row0 + rows - 1) / a.group + 1);
    const int all_iters = (span.n + BK - 1) / BK;
    const int it0 = static_cast<int>(static_cast<long long>(all_iters) * split / splits);
    const int it1 = static_cast<int>(static_cast<long long>(all_iters) * (split + 1) / splits);
    const int iters = it1 - it0;

    uint8_t* smem = tile_smem_raw + ((1024u - (smem_u32(tile_smem_raw) & 1023u)) & 1023u);
    const uint32_t sq = smem_u32(smem), sop = sq + 2 * G::kQ, sraw = sop + G::kStages * G::kOp;
    uint8_t* meta_base = smem + 2 * G::kQ + G::kStages * G::kOp + G::kRawStages * G::kRaw;
    volatile int* dead = &s_dead;

    if (warp == 12) {
        tmem_alloc(&s_tmem, 512);
        if (lane == 0) {
            mbar_init(&bars.q_full, 128);
            for (int s = 0; s < G::kStages; ++s) {
                mbar_init(&bars.full[s], 128);
                mbar_init(&bars.empty[s], 1);
            }
            for (int s = 0; s < kMetaSlots; ++s) mbar_init(&bars.meta[s], 128);
            for (int t = 0; t < 2; ++t) {
                mbar_init(&bars.s_full[t], 1);
                mbar_init(&bars.p_ready[t][0], 128);
                mbar_init(&bars.p_ready[t][1], 128);
                mbar_init(&bars.o_done[t], 1);
            }
            fence_mbar_init();
        }
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    if (warp >= 12) {
        // =============================== issuer ===============================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        // The whole warp runs the loop and one lane issues: control and addresses stay uniform over the warp, so
        // they live in uniform registers, as the instructions want them (from one lane's own registers each
        // MMA cost about 90 cycles to issue, and a pair of tiles 5400 cycles instead of 4250).
        const int n_iters = __shfl_sync(0xffffffffu, iters, 0);
        const bool both = __shfl_sync(0xffffffffu, static_cast<int>(two), 0) != 0;
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        if (warp == 12 && n_iters > 0) {
            constexpr uint32_t id_qk = tc_idesc<T>(BK, false);
            constexpr uint32_t id_pv = tc_idesc<T>(I8 ? 64 : D, true);
            uint32_t lead;
            asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(lead));
            auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, tile_wait(bar, parity, dead)) != 0; };
            auto stage = [&](int n) { return sop + (n % G::kStages) * G::kOp; };
            auto wait_full = [&](int n) { return wait(&bars.full[n % G::kStages], (n / G::kStages) & 1); };
            auto scores = [&](int t, int i) {
                const uint32_t d = tm + t * 128;
                const uint64_t q = sw128_desc(sq + t * G::kQ, 16, 1024), k = sw128_desc(stage(2 * i), 16, 1024);
                if (lead) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint64_t dq = q + (((kk >> 2) * (kTileRows * 128) + (kk & 3) * 32) >> 4);
                        const uint64_t dk = k + (((kk >> 2) * (BK * 128) + (kk & 3) * 32) >> 4);
                        // int8: every 64-dim block its own accumulator
                        tc_mma_ss(d + (I8 ? (kk >> 2) * BK : 0), dq, dk, id_qk, I8 ? (kk & 3) > 0 : kk > 0);
                    }
                    tc_commit(&bars.s_full[t]);
                }
                __syncwarp();
            };
            // half `part` of the tile's keys (int8: block `part` of the dims)
            auto outputs = [&](int t, int i, int part) {
                const uint32_t p = tm + t * 128, d = tm + 256 + t * 128;
                const uint64_t v = sw128_desc(stage(2 * i + 1), BK * 128, 1024);
                if (lead) {
                    if constexpr (!I8) {
#pragma unroll
                        for (int k = 0; k < BK / 32; ++k) {
                            const int ks = part * (BK / 32) + k;
                            tc_mma_ts(d, p + ks * 8, v + ((ks * 2048) >> 4), id_pv, i > 0 || ks > 0);
                        }
                    } else if (part < NH) {
#pragma unroll
                        for (int ks = 0; ks < BK / 16; ++ks)
                            tc_mma_ts(d + part * 64, p + part * (BK / 2) + ks * 8, v + ((part * (BK * 128) + ks * 2048) >> 4), id_pv,
                                      i > 0 || ks > 0);
                    }
                }
                __syncwarp();
            };
            auto commit = [&](uint64_t* bar) {
                if (lead) tc_commit(bar);
                __syncwarp();
            };
            bool ok = wait(&bars.q_full, 0) && wait_full(0);
            if (ok) {
                tc_fence_after();
                scores(0, 0);
                if (both) scores(1, 0);
                commit(&bars.empty[0]);
            }
            for (int i = 0; ok && i < n_iters; ++i) {
                const bool more = i + 1 < n_iters;
                ok = wait_full(2 * i + 1);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (t == 1 && !both) break;
#pragma unroll
                    for (int part = 0; part < 2; ++part) {
                        ok = ok && wait(&bars.p_ready[t][part], i & 1);
                        if (!ok) break;
                        tc_fence_after();
                        outputs(t, i, part);
                    }
                    if (!ok) break;
                    if (more) {
                        if (t == 0) ok = wait_full(2 * i + 2);
                        if (!ok) break;
                        tc_fence_after();
                        scores(t, i + 1);
                    } else {
                        commit(&bars.o_done[t]);
                    }
                }
                if (!ok) break;
                commit(&bars.empty[(2 * i + 1) % G::kStages]);
                if (more) commit(&bars.empty[(2 * i + 2) % G::kStages]);
            }
        }
        __syncwarp();
    } else if (warp >= 8) {
        // =============================== loaders ===============================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        const int lt = tid - 256, lw = warp - 8;
        const int piece = lt & 7;  // 16-byte piece of a 128-byte row
        const int32_t* tab = a.table + req * a.table_stride;
        // this warp's keys of a tile are KW consecutive ones; lane l looks up the l % KW-th of them
        constexpr int KW = BK / 4;
        const int my_key = KW * lw + lane % KW;
        auto lookup = [&](int it) {
            const int u = it * BK + my_key;
            if (it >= it1 || u >= span.n) return -1;
            const int pg = tab[a.c.page.div(span.key(u))];
            return pg < a.c.n_pages ? pg : -1;
        };
        int pg = lookup(it0);
        // ---- Q: rows lt / 8 + 16 j of both tiles ----
#pragma unroll 4
        for (int j = 0; j < (two ? kUnitRows : kTileRows) / 16; ++j) {
            const int row = (lt >> 3) + 16 * j;
            const int rr = row0 + row, i = a.by_group.div(rr);
            const bool live = row < rows;
            const T* qp = static_cast<const T*>(a.q) +
                          (live ? (r.first + i) * a.q_token_stride + (h * a.group + rr - i * a.group) * a.q_head_stride + piece * 8 : 0);
            const int tr = row & (kTileRows - 1);
            const uint32_t dst = sq + (row >> 7) * G::kQ + tr * 128 + ((piece ^ (tr & 7)) << 4);
#pragma unroll
            for (int b = 0; b < NH; ++b) cp_async_n<16>(dst + b * (kTileRows * 128), qp + (live ? 64 * b : 0), live ? 16 : 0);
        }
        cp_async_commit();
        auto offset_of = [&](int it, int pg, int* in_page) {
            const int j = span.key(it * BK + my_key);
            *in_page = pg >= 0 ? j - a.c.page.div(j) * a.c.page.d : 0;
            return pg >= 0 ? pg * a.c.page_stride + *in_page * a.c.token_stride + h * a.c.head_stride : -1ll;
        };
        bool ok = true;
        if constexpr (!I8) {
            // K and V tiles in turn, two copy groups in flight before the older one is handed over
            auto copy_tile = [&](const void* base, long long off, int n) {
                const uint32_t st = sop + (n % G::kStages) * G::kOp;
#pragma unroll
                for (int q = 0; q < KW / 4; ++q) {
                    const int row = KW * lw + 4 * q + (lane >> 3);
                    const long long o = __shfl_sync(0xffffffffu, off, 4 * q + (lane >> 3));
                    const T* src = static_cast<const T*>(base) + (o < 0 ? 0 : o + piece * 8);
                    const uint32_t dst = st + row * 128 + ((piece ^ (row & 7)) << 4);
#pragma unroll
                    for (int b = 0; b < NH; ++b) cp_async_n<16>(dst + b * (BK * 128), src + (o < 0 ? 0 : 64 * b), o >= 0 ? 16 : 0);
                }
                cp_async_commit();
            };
            for (int n = 0; n < 2 * iters && ok; n += 2) {
                const int i = n >> 1;
                int in_page;
                const long long off = offset_of(it0 + i, pg, &in_page);
                const uint32_t have = __ballot_sync(0xffffffffu, off >= 0);
                const int nx = lookup(it0 + i + 1);
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    const int m = n + kv;
                    if (m >= G::kStages && !tile_wait(&bars.empty[m % G::kStages], (m / G::kStages - 1) & 1, dead)) ok = false;
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    if (kv == 0) {
                        // the slot's last reader finished two key tiles ago
                        reinterpret_cast<uint32_t*>(meta_base + (i % kMetaSlots) * G::kMeta)[lw] = have;
                        mbar_arrive(&bars.meta[i % kMetaSlots]);
                    }
                    copy_tile(kv ? a.c.v : a.c.k, off, m);
                    cp_async_wait<1>();  // all but the copy just issued
                    fence_proxy_async_smem();
                    if (m == 0) mbar_arrive(&bars.q_full);
                    else mbar_arrive(&bars.full[(m - 1) % G::kStages]);
                }
                pg = nx;
            }
            cp_async_wait<0>();
            fence_proxy_async_smem();
            if (ok && iters > 0) mbar_arrive(&bars.full[(2 * iters - 1) % G::kStages]);
        } else {
            // Codes and scales go through a strip of a ring of each thread's own: it converts the pieces
            // that it copied, so only its own copies have to have arrived.
            constexpr int kPieces = D / 16;              // 16-byte pieces of a key's codes
            constexpr int kPer = 32 / kPieces;           // keys of a pass of the warp
            constexpr int kPass = KW / kPer;
            const int cp = lane % kPieces, cr = lane / kPieces;
            auto raw_at = [&](int i, int kv, int p) {
                return sraw + (i % G::kRawStages) * G::kRaw + ((kv * kPass + p) * 128 + lt) * 16;
            };
            auto raw_tail = [&](int i) { return sraw + (i % G::kRawStages) * G::kRaw + G::kRawCodes + lt * 16; };
            auto issue = [&](int i, int pg) {
                if (i < iters) {
                    int in_page;
                    const long long off = offset_of(it0 + i, pg, &in_page);
                    const uint32_t have = __ballot_sync(0xffffffffu, off >= 0);
#pragma unroll
                    for (int p = 0; p < kPass; ++p) {
                        const long long o = __shfl_sync(0xffffffffu, off, kPer * p + cr);
                        const long long src = o < 0 ? 0 : o + cp * 16;
                        cp_async_n<16>(raw_at(i, 0, p), static_cast<const int8_t*>(a.c.k) + src, o >= 0 ? 16 : 0);
                        cp_async_n<16>(raw_at(i, 1, p), static_cast<const int8_t*>(a.c.v) + src, o >= 0 ? 16 : 0);
                    }
                    // lanes 0-15: the K scales of their key, 16-31: the V scales; lane 0 keeps which keys exist
                    const long long sb = pg >= 0 ? ((static_cast<long long>(pg) * a.c.page.d + in_page) * a.c.kv_heads + h) * NH : 0;
                    cp_async_n<4 * NH>(raw_tail(i), (lane < 16 ? a.c.ks : a.c.vs) + sb, pg >= 0 ? 4 * NH : 0);
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(raw_tail(i) + 8), "r"(have & 0xffffu) : "memory");
                }
                cp_async_commit();
            };
            for (int s = 0; s < G::kRawStages; ++s) {
                const int nx = lookup(it0 + s + 1);
                issue(s, pg);
                pg = nx;
            }
            for (int i = 0; i < iters && ok; ++i) {
                for (int kv = 0; kv < 2; ++kv) {
                    const int m = 2 * i + kv;
                    if (m >= G::kStages && !tile_wait(&bars.empty[m % G::kStages], (m / G::kStages - 1) & 1, dead)) ok = false;
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    if (kv == 0) {
                        cp_async_wait<G::kRawStages - 1>();
                        // the meta slot's last reader finished two key tiles ago
                        uint8_t* mt = meta_base + (i % kMetaSlots) * G::kMeta;
                        float* dst = reinterpret_cast<float*>(mt + 16) + (lane < 16 ? 0 : BK * NH) + (KW * lw + (lane & 15)) * NH;
#pragma unroll
                        for (int b = 0; b < NH; ++b) dst[b] = ldsf(raw_tail(i) + 4 * b);
                        if (lane == 0) reinterpret_cast<unsigned short*>(mt)[lw] = static_cast<unsigned short>(lds32(raw_tail(i) + 8));
                        mbar_arrive(&bars.meta[i % kMetaSlots]);
                    }
                    const uint32_t st = sop + (m % G::kStages) * G::kOp;
#pragma unroll
                    for (int p = 0; p < kPass; ++p) {
                        const int row = KW * lw + kPer * p + cr;
                        const uint4 w = lds128(raw_at(i, kv, p));
                        uint32_t x[8];
                        codes_to_pairs_as<T>(w.x, x[0], x[1]);
                        codes_to_pairs_as<T>(w.y, x[2], x[3]);
                        codes_to_pairs_as<T>(w.z, x[4], x[5]);
                        codes_to_pairs_as<T>(w.w, x[6], x[7]);
                        const uint32_t dst = st + (cp >> 2) * (BK * 128) + row * 128;
                        // the two halves of the row start with different pieces: no bank conflict
                        const int swap = cp >> 2, pc = (cp & 3) * 2;
                        const uint32_t d0 = dst + (((pc + swap) ^ (row & 7)) << 4), d1 = dst + (((pc + 1 - swap) ^ (row & 7)) << 4);
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(d0), "r"(swap ? x[4] : x[0]),
                                     "r"(swap ? x[5] : x[1]), "r"(swap ? x[6] : x[2]), "r"(swap ? x[7] : x[3])
                                     : "memory");
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(d1), "r"(swap ? x[0] : x[4]),
                                     "r"(swap ? x[1] : x[5]), "r"(swap ? x[2] : x[6]), "r"(swap ? x[3] : x[7])
                                     : "memory");
                    }
                    fence_proxy_async_smem();
                    if (m == 0) mbar_arrive(&bars.q_full);  // Q's copies are older than the codes'
                    mbar_arrive(&bars.full[m % G::kStages]);
                }
                const int nx = lookup(it0 + i + G::kRawStages + 1);
                issue(i + G::kRawStages, pg);
                pg = nx;
            }
            cp_async_wait<0>();
        }
    } else {
        // =============================== softmax ===============================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int t = warp >> 2, row = tid & 127;
        if (t == 0 || two) {
            const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
            const uint32_t ts = tmem + lane_base + t * 128, to = tmem + lane_base + 256 + t * 128;
            const int rr = row0 + t * kTileRows + row;
            const bool live = t * kTileRows + row < rows;
            const int tok = rr / a.group;
            const int p = r.len - r.n + tok;
            // This row sees the virtual keys u_low .. u_high and those below u_sink.  Key tiles between t_low
            // and t_high need no mask: seen whole by every row of the tile.
            int u_low = 0, u_high = 0x7ffffffe, u_sink = 0, t_low = 0, t_high = 0x7ffffffe;
            if (a.causal) {
                const int shift = span.sunk - span.lo;  // from keys to virtual keys
                const int p_first = r.len - r.n + (row0 + t * kTileRows) / a.group;
                const int p_last = r.len - r.n + (row0 + min(rows, (t + 1) * kTileRows) - 1) / a.group;
                u_high = p < 0 ? -1 : p + shift;
                t_high = p_first < 0 ? -1 : p_first + shift;
                if (a.window > 0) {
                    u_low = max(window_low(a, p) + shift, 0);
                    t_low = max(window_low(a, p_last) + shift, 0);
                    u_sink = a.sinks;
                }
            }
            float m_ref = -INFINITY, l = 0.0f;
            constexpr bool kHalf = std::is_same<T, __half>::value, kUnits = I8 && kHalf;
            // log2 of how far a weight may pass 2^kLift, and of the weight at the maximum that m_ref was taken
            // from: together below fp16's 65504 (int8: times a V scale over its unit, below 2)
            constexpr float kSlack = kHalf ? 3.0f : 8.0f, kLift = !kHalf ? 0.0f : (I8 ? 11.0f : 12.0f);
            float unit[NH];
#pragma unroll
            for (int b = 0; b < NH; ++b) unit[b] = 0.0f;
            bool ok = true;
            for (int i = 0; i < iters; ++i) {
                const uint8_t* mt = meta_base + (i % kMetaSlots) * G::kMeta;
                ok = tile_wait(&bars.meta[i % kMetaSlots], (i / kMetaSlots) & 1, dead) &&
                     tile_wait(&bars.s_full[t], i & 1, dead);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                // ---- scores ----
                float s[BK];
                if constexpr (!I8) {
                    uint32_t v[BK / 32][32];
#pragma unroll
                    for (int c = 0; c < BK / 32; ++c) tmem_ld32(ts + 32 * c, v[c]);
                    tc_wait_ld();
#pragma unroll
                    for (int c = 0; c < BK / 32; ++c) {
                        reg_fence32(v[c]);
#pragma unroll
                        for (int k = 0; k < 32; ++k) s[32 * c + k] = __uint_as_float(v[c][k]);
                    }
                } else {
                    const float* ks = reinterpret_cast<const float*>(mt + 16);
#pragma unroll
                    for (int c0 = 0; c0 < BK; c0 += 32) {
                        uint32_t v[NH][32];
#pragma unroll
                        for (int b = 0; b < NH; ++b) tmem_ld32(ts + b * BK + c0, v[b]);
                        tc_wait_ld();
#pragma unroll
                        for (int b = 0; b < NH; ++b) reg_fence32(v[b]);
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            float x = __uint_as_float(v[0][k]) * ks[(c0 + k) * NH];
                            if constexpr (NH == 2) x = fmaf(__uint_as_float(v[1][k]), ks[(c0 + k) * NH + 1], x);
                            s[c0 + k] = x;
                        }
                    }
                }
                // ---- mask: keys k with k_low <= k <= k_high, or k below the sinks; those that exist ----
                const int u0 = (it0 + i) * BK;
                const uint32_t* have = reinterpret_cast<const uint32_t*>(mt);
                uint32_t all_here = 0xffffffffu;
#pragma unroll
                for (int w = 0; w < BK / 32; ++w) all_here &= have[w];
                const bool clear = all_here == 0xffffffffu && u0 + BK - 1 <= t_high && u0 >= t_low;
                if (!clear) {
                    const int k_high = u_high - u0, k_low = u_low - u0, k_sink = u_sink - u0;
                    auto below = [](int n) { return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1); };
#pragma unroll
                    for (int w = 0; w < BK / 32; ++w) {
                        const uint32_t m = have[w] & below(k_high + 1 - 32 * w) & (~below(k_low - 32 * w) | below(k_sink - 32 * w));
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (!(m >> k & 1u)) s[32 * w + k] = -INFINITY;
                    }
                }
                // ---- running maximum: moved when it grows by more than 2^kSlack ----
                float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int k = 4; k < BK; k += 8) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mx[j] = k + j + 4 < BK ? fmaxf(fmaxf(mx[j], s[k + j]), s[k + j + 4]) : fmaxf(mx[j], s[k + j]);
                }
                const float top = fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), a.scale_log2, -kLift);
                float alpha = 1.0f;
                const bool grow = top > m_ref + kSlack || (m_ref == -INFINITY && top > -INFINITY);
                if (grow) {
                    alpha = m_ref == -INFINITY ? 0.0f : ex2(m_ref - top);
                    m_ref = top;
                }
                float f[NH];
#pragma unroll
                for (int b = 0; b < NH; ++b) f[b] = alpha;
                bool rescale = grow;
                if constexpr (kUnits) {
                    const float* vs = reinterpret_cast<const float*>(mt + 16) + BK * NH;
#pragma unroll
                    for (int b = 0; b < NH; ++b) {
                        float vm = 0.0f;
                        for (int k = 0; k < BK; ++k) vm = fmaxf(vm, vs[k * NH + b]);
                        vm = __uint_as_float(__float_as_uint(vm) & 0x7f800000u);
                        if (vm > unit[b]) {
                            f[b] *= unit[b] / vm;
                            unit[b] = vm;
                            rescale = true;
                        }
                    }
                }
                if (i > 0 && __any_sync(0xffffffffu, rescale)) {
                    // the previous product into O is complete: this tile's S was issued after it
#pragma unroll
                    for (int c0 = 0; c0 < D; c0 += 32) {
                        uint32_t v[32];
                        tmem_ld32(to + c0, v);
                        tc_wait_ld();
                        reg_fence32(v);
#pragma unroll
                        for (int k = 0; k < 32; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * f[c0 / 64]);
                        tmem_st32(to + c0, v);
                    }
                }
                // ---- weights, two at a time where the arithmetic is packed ----
                const float base = m_ref == -INFINITY ? 0.0f : m_ref;
                const uint64_t scale2 = pack_f32x2(a.scale_log2, a.scale_log2), base2 = pack_f32x2(-base, -base);
                uint64_t sum2[2] = {0, 0};
                auto weight = [&](int k) {  // elements k and k + 1
                    float x, y;
                    unpack_f32x2(fma_f32x2(pack_f32x2(s[k], s[k + 1]), scale2, base2), x, y);
                    s[k] = ex2(x);
                    s[k + 1] = ex2(y);
                    sum2[k >> 1 & 1] = add_f32x2(sum2[k >> 1 & 1], pack_f32x2(s[k], s[k + 1]));
                };
                if constexpr (!I8) {
#pragma unroll
                    for (int part = 0; part < 2; ++part) {
                        uint32_t v[32];
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            weight(64 * part + 2 * k);
                            v[k] = pack2<T>(s[64 * part + 2 * k], s[64 * part + 2 * k + 1]);
                        }
                        tmem_st32(ts + 32 * part, v);
                        tc_wait_st();
                        tc_fence_before();
                        mbar_arrive(&bars.p_ready[t][part]);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < BK; k += 2) weight(k);
                    const float* vs = reinterpret_cast<const float*>(mt + 16) + BK * NH;
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        if (b < NH) {
                            float inv = 1.0f;
                            if constexpr (kUnits) inv = unit[b < NH ? b : 0] > 0.0f ? 1.0f / unit[b < NH ? b : 0] : 0.0f;
                            uint32_t v[32];
#pragma unroll
                            for (int k = 0; k < 32; ++k) {
                                float x0 = vs[2 * k * NH + b], x1 = vs[(2 * k + 1) * NH + b];
                                if constexpr (kUnits) {
                                    x0 *= inv;
                                    x1 *= inv;
                                }
                                v[k] = pack2<T>(s[2 * k] * x0, s[2 * k + 1] * x1);
                            }
                            tmem_st32(ts + b * (BK / 2), v);
                        }
                        tc_wait_st();
                        tc_fence_before();
                        mbar_arrive(&bars.p_ready[t][b]);
                    }
                }
                float x0, x1;
                unpack_f32x2(add_f32x2(sum2[0], sum2[1]), x0, x1);
                l = fmaf(l, alpha, x0 + x1);
            }
            if (iters > 0 && ok) ok = tile_wait(&bars.o_done[t], 0, dead);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            if (ok) {
                // parts that only the other blocks have
                if (a.parts_ml && live && split == 0)
                    for (int i = splits; i < a.splits; ++i)
                        a.parts_ml[i * static_cast<long long>(a.tokens) * a.heads + static_cast<long long>(r.first + tok) * a.heads +
                                   h * a.group + (rr - tok * a.group)] = make_float2(-INFINITY, 0.0f);
                const long long qh = static_cast<long long>(r.first + tok) * a.heads + h * a.group + (rr - tok * a.group);
                // Rows go out through this warp's part of the Q tile (free: the last product is done), so that a warp
                // writes whole rows and not 32 of them 16 bytes at a time.
                const uint32_t rows_at = sq + t * G::kQ + (warp & 3) * 32 * (D * 2);
                const bool staged = !a.parts_acc && iters > 0;  // without a product Q's copies may still be landing
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                if (staged && live && a.lse) a.lse[qh] = l == 0.0f ? -INFINITY : (m_ref + log2f(l)) * kLn2;
#pragma unroll
                for (int c0 = 0; c0 < D; c0 += 32) {
                    float acc[32];
                    if (iters > 0) {
                        uint32_t v[32];
                        tmem_ld32(to + c0, v);
                        tc_wait_ld();
                        reg_fence32(v);
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            acc[k] = __uint_as_float(v[k]);
                            if constexpr (kUnits) acc[k] *= unit[c0 / 64];
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; ++k) acc[k] = 0.0f;
                    }
                    if (staged) {
#pragma unroll
                        for (int k = 0; k < 32; ++k) acc[k] = l == 0.0f ? 0.0f : acc[k] * inv;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int pc = c0 / 8 + k;  // piece of 16 bytes, permuted by the row
                            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(rows_at + lane * (D * 2) + ((pc ^ (lane & 7)) << 4)),
                                         "r"(pack2<T>(acc[8 * k], acc[8 * k + 1])), "r"(pack2<T>(acc[8 * k + 2], acc[8 * k + 3])),
                                         "r"(pack2<T>(acc[8 * k + 4], acc[8 * k + 5])), "r"(pack2<T>(acc[8 * k + 6], acc[8 * k + 7]))
                                         : "memory");
                        }
                    } else if (live) {
                        attention_store<T, 32>(a, split, qh, D, c0, c0 == 0, acc, m_ref, l);
                    }
                }
                if (staged) {
                    __syncwarp();
                    constexpr int kRowPieces = D / 8;
                    const int first = t * kTileRows + (warp & 3) * 32;
#pragma unroll 4
                    for (int j = 0; j < kRowPieces; ++j) {
                        const int idx = j * 32 + lane, wr = idx / kRowPieces, pc = idx % kRowPieces;
                        if (first + wr >= rows) continue;
                        const int r2 = row0 + first + wr, t2 = a.by_group.div(r2);
                        const long long q2 = static_cast<long long>(r.first + t2) * a.heads + h * a.group + (r2 - t2 * a.group);
                        *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + q2 * D + pc * 8) =
                            lds128(rows_at + wr * (D * 2) + ((pc ^ (wr & 7)) << 4));
                    }
                }
                tc_fence_before();
            }
        }
    }
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Rows whose keys were split, joined from their parts: 8 dims per thread, parts in order.  (Joined instead in
// the few-rows kernel's store, the 12 parts of a shared prefix cost it 36 of 103 us: three rows of a unit
// leave most of a CTA waiting for their loads.)
template <typename T, int D>
__global__ void __launch_bounds__(256) k_attention_join(const AttnPagedArgs a) {
    constexpr int DP = D / 16 < 8 ? 8 : D / 16;  // dims per thread
    constexpr int kPer = D / DP;                 // threads per row
    const long long qh = static_cast<long long>(blockIdx.x) * (256 / kPer) + threadIdx.x / kPer;
    if (qh >= static_cast<long long>(a.tokens) * a.heads) return;
    const int tok = static_cast<int>(qh / a.heads);
    if (a.cu) {
        // only rows that the many-rows kernel took
        if (tok < a.cu[0] || tok >= a.cu[a.n_req]) return;
        const ReqRows r = request_rows(a, last_not_above(a.cu, a.n_req, tok));
        if (r.n * a.group <= a.small_rows) return;
    }
    float acc[DP];
#pragma unroll
    for (int d = 0; d < DP; ++d) acc[d] = 0.0f;
    const int lane = threadIdx.x % kPer, d0 = lane * DP;
    const long long rows = static_cast<long long>(a.tokens) * a.heads;
    float mx = -INFINITY, sum = 0.0f;
    // the parts, a few loads at once
    constexpr int kBatch = 4;
    for (int i0 = 0; i0 < a.n_parts; i0 += kBatch) {
        float2 ml[kBatch];
        float4 v[kBatch][DP / 4];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const long long at = min(i0 + k, a.n_parts - 1) * rows + qh;
            ml[k] = a.parts_ml[at];
            if (i0 + k >= a.n_parts) ml[k] = make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int d = 0; d < DP / 4; ++d) v[k][d] = *reinterpret_cast<const float4*>(a.parts_acc + at * D + d0 + 4 * d);
        }
        const float own = mx;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) mx = fmaxf(mx, ml[k].x);
        const float base = mx == -INFINITY ? 0.0f : mx;
        const float f = ex2(own - base);
        sum = sum == 0.0f ? 0.0f : sum * f;
#pragma unroll
        for (int d = 0; d < DP; ++d) acc[d] = sum == 0.0f ? 0.0f : acc[d] * f;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            if (ml[k].y == 0.0f) continue;  // that part saw no key (its output is not written)
            const float w = ex2(ml[k].x - base);
            sum = fmaf(ml[k].y, w, sum);
#pragma unroll
            for (int d = 0; d < DP / 4; ++d) {
                acc[4 * d] = fmaf(v[k][d].x, w, acc[4 * d]);
                acc[4 * d + 1] = fmaf(v[k][d].y, w, acc[4 * d + 1]);
                acc[4 * d + 2] = fmaf(v[k][d].z, w, acc[4 * d + 2]);
                acc[4 * d + 3] = fmaf(v[k][d].w, w, acc[4 * d + 3]);
            }
        }
    }
    attention_store<T, DP>(a, 0, qh, D, d0, lane == 0, acc, mx, sum, true);
}

}  // namespace asdsl
