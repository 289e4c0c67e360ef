// Attention of many query rows per key head (chunks of prompts, frames): tcgen05 matrix products over KV tiles of 128 keys.
//
// A work item is 256 query rows of one (sequence, key head), as two tiles A and B of 128 rows.  Per KV tile and row tile
//     S = Q K^T (tensor memory, fp32)  ->  P = 2^(c (S - m)) (16 bits, over S in tensor memory)  ->  O += P V.
// One warp fetches pages by TMA into a ring of K and V tiles, one issues the products, and four each own the softmax of
// A and of B, one thread per row, so that row maxima and sums need no exchange.  While A's weights are computed the tensor
// core works on B.  The running maximum moves only when a row has outgrown it by 2^8 (weights stay below 2^8, exact in the
// quotient), so O in tensor memory is rescaled rarely.
// Keys stay K-major as they lie in the page, values are read in the same layout as the MN-major operand: nothing is
// transposed.  Rows of V outside the sequence are zeroed in shared memory before their product, since 0 x NaN is no zero.
#include <cuda.h>

#include <mutex>

#include "paged_attention.cuh"

namespace b200 {
namespace {

constexpr int kChunkThreads = 384;  // three warpgroups; warps 10 and 11 only fill the third
// registers a thread: 384 x 168 at launch = 64512 >= 256 x 208 + 128 x 80 = 63488
constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;
constexpr int kChunkRows = 256;   // two row tiles
constexpr int kKeyTile = 128;
constexpr int kSlabBytes = 128 * 128;  // 128 rows of 64 16-bit elements, 128-byte swizzle
constexpr float kLazyRescale = 8.0f;   // log2 of how far a weight may exceed one

template <int D>
struct ChunkCfg {
    static constexpr int kTileBytes = D / 64 * kSlabBytes;
    static constexpr int kStages = D == 128 ? 5 : 8;
    static constexpr int kSmemBytes = (2 + kStages) * kTileBytes + 1024 + 256;
    static constexpr int kWarpPartial = 32 * (D + 2);  // floats: 32 rows x D, maxima, sums
};

// 64-bit operand descriptor of a tile whose rows of 128 bytes run along N (MN-major, 128-byte swizzle): groups of 8 K rows
// are 1024 bytes apart, blocks of 64 elements of N one slab.
__device__ __forceinline__ uint64_t smem_desc_mn128(uint32_t addr) {
    uint64_t d = 0;
    d |= (uint64_t)((addr >> 4) & 0x3FFFu);
    d |= (uint64_t)(kSlabBytes >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void *map, uint64_t *bar, int c0, int c1, int c2, int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}

template <typename T>
struct IsBf16 {
    static constexpr uint32_t value = 0;
};
template <>
struct IsBf16<__nv_bfloat16> {
    static constexpr uint32_t value = 1;
};
// fp32 accumulators, A and B of type T, M = 128; bit 16: B is MN-major.
template <typename T>
__host__ __device__ constexpr uint32_t idesc_f16(int n, uint32_t b_mn_major) {
    return (1u << 4) | (IsBf16<T>::value << 7) | (IsBf16<T>::value << 10) | (b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(128 >> 4) << 24);
}

struct ChunkExtra {
    int page_box;  // tokens per TMA box: min(page_tokens, 128)
    unsigned long long wait_limit_ns;
    int debug_drop_load;
};

template <typename T, int D>
__global__ void __launch_bounds__(kChunkThreads, 1)
    attention_chunk_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                           const AttnParams a, const ChunkExtra ex) {
    using C = ChunkCfg<D>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ PlanShared<kChunkThreads> plan;
    __shared__ Item items[10];  // every warp's own place in the plan, kept out of the loops' registers
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *ring = smem + 2 * C::kTileBytes;
    uint64_t *kv_full = reinterpret_cast<uint64_t *>(ring + C::kStages * C::kTileBytes);
    uint64_t *kv_empty = kv_full + C::kStages;
    uint64_t *q_ready = kv_empty + C::kStages;  // [2] the row tile's queries are in shared memory
    uint64_t *s_full = q_ready + 2;             // [2] scores are in tensor memory
    uint64_t *p_ready = s_full + 2;             // [2] weights are in tensor memory, O is rescaled
    uint64_t *o_full = p_ready + 2;             // [2] the last product of a run has landed
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(o_full + 2);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const WaitCtx wctx{abort_flag, a.c.status, ex.wait_limit_ns};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    pdl_trigger();
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&kv_full[s], 1);
            mbar_init(&kv_empty[s], 1);
        }
        for (int x = 0; x < 2; ++x) {
            mbar_init(&q_ready[x], 4);
            mbar_init(&s_full[x], 1);
            mbar_init(&p_ready[x], 4);
            mbar_init(&o_full[x], 1);
        }
        *abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
    }
    pdl_wait();
    long long total, x0, x1;
    int runs;
    {
        Item first;
        if (!plan_run<kChunkRows, kKeyTile, kChunkThreads>(a, plan, total, runs, x0, x1, first)) return;
        if (lane == 0 && warp < 10) items[warp] = first;
    }
    Item &it = items[min(warp, 9)];
    if (warp == 9) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    const uint32_t tmem_o = tmem + 2 * kKeyTile;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == 8) {
            // ---- pages -> ring.  Tile order K0 V0 K1 V1 ...; lanes issue a box each.
            int s = 0;
            uint32_t ph = 0;
            bool ok = true, drop = ex.debug_drop_load != 0;
            const int boxes = kKeyTile / ex.page_box;  // along the keys of a tile
            for (long long x = x0; ok && x < x1;) {
                const long long end = it.begin + (it.kt1 - it.kt0);
                const int kt0 = it.kt0 + (int)(x - it.begin), kt1 = it.kt0 + (int)(min(x1, end) - it.begin);
                const int lo = it.lo, hi = it.hi, kv_head = it.h;
                const int *table = a.c.page_table + (long long)it.s * a.c.max_pages;
                for (int kt = kt0; ok && kt < kt1; ++kt) {
                    // lane b holds the page of box b (at most 8 boxes)
                    const int key = kt * kKeyTile + lane * ex.page_box;
                    const bool live = lane < boxes && key < hi && key + ex.page_box > lo;
                    int page = 0;
                    if (live) {
                        page = table[key >> a.c.page_shift];
                        if (page < 0 || page >= a.c.n_pages) {
                            report_bad_page(a.c);
                            page = a.c.n_pages;  // outside the tensor map: zeros arrive
                        }
                    }
                    const int token = key & ((1 << a.c.page_shift) - 1);
                    const unsigned mask = __ballot_sync(0xffffffffu, live);
                    const uint32_t bytes = (uint32_t)__popc(mask) * (uint32_t)ex.page_box * (D * 2);
                    for (int kv = 0; kv < 2; ++kv) {
                        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&kv_empty[s], ph ^ 1u, wctx, KS_TIMEOUT_SMEM_EMPTY));
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(&kv_full[s], bytes);
                        __syncwarp();
                        if (live && !drop) {
                            const uint32_t dst = smem_u32(ring + s * C::kTileBytes) + (uint32_t)(lane * ex.page_box * 128);
#pragma unroll
                            for (int d = 0; d < D / 64; ++d)
                                tma_load_4d(dst + d * kSlabBytes, kv ? &tm_v : &tm_k, &kv_full[s], d * 64, token, kv_head, page);
                        }
                        drop = false;
                        if (++s == C::kStages) { s = 0; ph ^= 1u; }
                    }
                }
                x = min(x1, end);
                if (x < x1) {
                    __syncwarp();
                    if (lane == 0) next_item<kChunkRows, kKeyTile>(a, it);
                    __syncwarp();
                }
            }
        } else if (warp == 9) {
            // ---- products
            constexpr uint32_t idesc_s = idesc_f16<T>(kKeyTile, 0), idesc_o = idesc_f16<T>(D, 1);
            int s = 0;
            uint32_t ph = 0, q_ph = 0, p_ph = 0;  // bit x: parity of the row tile's barrier
            bool ok = true;
            auto wait = [&](uint64_t *bar, uint32_t parity, int code) {
                ok = ok && __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, wctx, code));
                return ok;
            };
            auto scores = [&](int x, int stage) {  // S_x = Q_x K^T, then s_full[x]
                if (lane == 0) {
                    const uint64_t qd = umma_smem_desc_k128(smem_u32(smem + x * C::kTileBytes));
                    const uint64_t kd = umma_smem_desc_k128(smem_u32(ring + stage * C::kTileBytes));
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint64_t off = (uint64_t)(((k / 4) * kSlabBytes + (k % 4) * 32) >> 4);
                        umma_f16_ss(tmem + x * kKeyTile, qd + off, kd + off, idesc_s, k != 0);
                    }
                    umma_commit(&s_full[x]);
                }
                __syncwarp();
            };
            for (long long x = x0; ok && x < x1;) {
                const long long end = it.begin + (it.kt1 - it.kt0);
                const int kt0 = it.kt0 + (int)(x - it.begin), kt1 = it.kt0 + (int)(min(x1, end) - it.begin);
                const int lo = it.lo, hi = it.hi;
                const int tiles = it.rows - it.rt * kChunkRows > 128 ? 2 : 1;
                for (int kt = kt0 - 1; ok && kt < kt1; ++kt) {
                    // V of tile kt and K of tile kt + 1 are the next two stages of the ring
                    const int vs = s;
                    if (kt >= kt0) {
                        if (!wait(&kv_full[s], ph, KS_TIMEOUT_SMEM_FULL)) break;
                        if (++s == C::kStages) { s = 0; ph ^= 1u; }
                        if (kt * kKeyTile < lo || (kt + 1) * kKeyTile > hi) {
                            uint8_t *v = ring + vs * C::kTileBytes;
                            for (int i = lane; i < kKeyTile * (D / 8); i += 32) {
                                const int row = i / (D / 8), c = i % (D / 8), key = kt * kKeyTile + row;
                                if (key < lo || key >= hi)
                                    *reinterpret_cast<uint4 *>(v + (c / 8) * kSlabBytes + row * 128 + (c % 8) * 16) =
                                        make_uint4(0, 0, 0, 0);
                            }
                            fence_proxy_async_smem();
                            __syncwarp();
                        }
                    }
                    const int ks = s;
                    if (kt + 1 < kt1) {
                        if (!wait(&kv_full[s], ph, KS_TIMEOUT_SMEM_FULL)) break;
                        if (++s == C::kStages) { s = 0; ph ^= 1u; }
                    }
                    for (int rtile = 0; rtile < tiles; ++rtile) {
                        if (kt >= kt0) {
                            if (!wait(&p_ready[rtile], (p_ph >> rtile) & 1u, KS_TIMEOUT_SOFTMAX)) break;
                            p_ph ^= 1u << rtile;
                            tc_fence_after_sync();
                            if (lane == 0) {
                                const uint64_t vd = smem_desc_mn128(smem_u32(ring + vs * C::kTileBytes));
#pragma unroll
                                for (int k = 0; k < kKeyTile / 16; ++k)
                                    umma_f16_ts(tmem_o + rtile * D, tmem + rtile * kKeyTile + k * 8,
                                                vd + (uint64_t)(k * (2048 >> 4)), idesc_o, kt != kt0 || k != 0);
                                if (kt + 1 == kt1) umma_commit(&o_full[rtile]);
                            }
                            __syncwarp();
                        } else {
                            if (!wait(&q_ready[rtile], (q_ph >> rtile) & 1u, KS_TIMEOUT_SMEM_FULL)) break;
                            q_ph ^= 1u << rtile;
                            tc_fence_after_sync();
                        }
                        // the products of one CTA execute in the order of their issue, so S_x is written over P_x only
                        // after the product that reads P_x
                        if (kt + 1 < kt1) scores(rtile, ks);
                    }
                    if (!ok) break;
                    if (lane == 0) {
                        if (kt >= kt0) umma_commit(&kv_empty[vs]);
                        if (kt + 1 < kt1) umma_commit(&kv_empty[ks]);
                    }
                    __syncwarp();
                }
                x = min(x1, end);
                if (x < x1) {
                    __syncwarp();
                    if (lane == 0) next_item<kChunkRows, kKeyTile>(a, it);
                    __syncwarp();
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        // ---- softmax: warps 0-3 own row tile A, 4-7 row tile B; a thread owns a row
        const int tile = warp >> 2, sub = warp & 3;
        const uint32_t lanes = (uint32_t)(sub * 32) << 16;
        const uint32_t ts = tmem + lanes + tile * kKeyTile, to = tmem_o + lanes + tile * D;
        uint32_t s_ph = 0, o_ph = 0;
        bool ok = true;
        for (long long x = x0; ok && x < x1;) {
            const long long end = it.begin + (it.kt1 - it.kt0);
            const int kt0 = it.kt0 + (int)(x - it.begin), kt1 = it.kt0 + (int)(min(x1, end) - it.begin);
            const int row0 = it.rt * kChunkRows + tile * 128;
            if (row0 < it.rows) {
                const int r = row0 + sub * 32 + lane;
                const bool live = r < it.rows;
                const int tok = live ? r / a.group : 0, head = it.h * a.group + (live ? r % a.group : 0);
                int lo = 0, hi = 0x7fffffff;  // a row that is not there masks nothing
                if (live) visible_keys(a, it.seq.keys - it.seq.n + tok, it.seq.keys, lo, hi);
                const int lo_max = __reduce_max_sync(0xffffffffu, lo), hi_min = __reduce_min_sync(0xffffffffu, hi);
                {  // the row's queries, in the swizzled K-major layout
                    const uint4 *src = reinterpret_cast<const uint4 *>(
                        reinterpret_cast<const T *>(a.q) + (long long)(it.seq.q0 + tok) * a.q_ts + head * a.q_hs);
                    const int rr = sub * 32 + lane;
                    uint8_t *dst = smem + tile * C::kTileBytes + rr * 128;
#pragma unroll
                    for (int c = 0; c < D / 8; ++c)
                        *reinterpret_cast<uint4 *>(dst + (c / 8) * kSlabBytes + (((c & 7) ^ (rr & 7)) << 4)) =
                            live ? src[c] : make_uint4(0, 0, 0, 0);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&q_ready[tile]);
                }
                float m = -INFINITY, l = 0.0f;
                for (int kt = kt0; kt < kt1; ++kt) {
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_full[tile], s_ph, wctx, KS_TIMEOUT_SOFTMAX));
                    if (!ok) break;
                    s_ph ^= 1u;
                    tc_fence_after_sync();
                    // scores are read twice, first for the maximum, then for the weights: 128 fp32 registers less, for
                    // 64 KB of tensor-memory reads per tile
                    const int key0 = kt * kKeyTile;
                    const bool edge = key0 < lo_max || key0 + kKeyTile > hi_min;
                    auto hide = [&](uint32_t(&s)[32], int c) {
                        if (!edge) return;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const int key = key0 + 32 * c + i;
                            if (key < lo || key >= hi) s[i] = 0xff800000u;
                        }
                    };
                    uint32_t s[2][32];
                    float top = -INFINITY;
                    tmem_ld_32x32(ts, s[0]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        tmem_ld_wait();
                        tmem_ld_32x32(ts + 32 * ((c + 1) & 3), s[(c + 1) & 1]);  // the last one is the first of the second pass
                        hide(s[c & 1], c);
                        float t4[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) t4[i] = __uint_as_float(s[c & 1][i]);
#pragma unroll
                        for (int i = 4; i < 32; ++i) t4[i & 3] = fmaxf(t4[i & 3], __uint_as_float(s[c & 1][i]));
                        top = fmaxf(top, fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])));
                    }
                    if (kt == kt0) {
                        m = top;
                    } else if (__any_sync(0xffffffffu, (top - m) * a.scale_log2 > kLazyRescale)) {
                        const float mn = fmaxf(m, top);
                        const float f = m == -INFINITY ? 0.0f : fast_ex2((m - mn) * a.scale_log2);
                        m = mn;
                        l *= f;
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t o[32];
                            tmem_ld_32x32(to + 32 * c, o);
                            tmem_ld_wait();
                            uint32_t u[2][16];
#pragma unroll
                            for (int i = 0; i < 32; ++i) u[i / 16][i % 16] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tmem_st_32x16(to + 32 * c, u[0]);
                            tmem_st_32x16(to + 32 * c + 16, u[1]);
                        }
                    }
                    const float ref = m == -INFINITY ? 0.0f : m * a.scale_log2;
                    float sum[4] = {};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        tmem_ld_wait();
                        if (c < 3) tmem_ld_32x32(ts + 32 * (c + 1), s[(c + 1) & 1]);
                        hide(s[c & 1], c);
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float e0 = fast_ex2(fmaf(__uint_as_float(s[c & 1][2 * i]), a.scale_log2, -ref));
                            const float e1 = fast_ex2(fmaf(__uint_as_float(s[c & 1][2 * i + 1]), a.scale_log2, -ref));
                            sum[(2 * i) & 3] += e0;
                            sum[(2 * i + 1) & 3] += e1;
                            w[i] = Half2Of<T>::pack(e0, e1);
                        }
                        // columns 16 c: scores that have been read already
                        tmem_st_32x16(ts + 16 * c, w);
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tmem_st_wait();
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_ready[tile]);
                }
                if (ok) {
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(&o_full[tile], o_ph, wctx, KS_TIMEOUT_TMEM_FULL));
                    o_ph ^= 1u;
                }
                if (!ok) break;
                tc_fence_after_sync();
                const int first = run_of(it.begin, total, runs), final = run_of(end - 1, total, runs);
                T *dst = reinterpret_cast<T *>(a.out) + (long long)(it.seq.q0 + tok) * a.o_ts + head * a.o_hs;
                if (first == final) {
                    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld_32x32(to + 32 * c, o);
                        tmem_ld_wait();
                        if (live) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                uint32_t p[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    p[e] = Half2Of<T>::pack(__uint_as_float(o[8 * i + 2 * e]) * inv,
                                                            __uint_as_float(o[8 * i + 2 * e + 1]) * inv);
                                *reinterpret_cast<uint4 *>(dst + 32 * c + 8 * i) = make_uint4(p[0], p[1], p[2], p[3]);
                            }
                        }
                    }
                } else {
                    // [slot of the CTA][warp]: columns in vectors of four, 32 rows each
                    auto part_of = [&](int cta) {
                        return a.partials + ((long long)(2 * cta + (cta == first ? 1 : 0)) * 8 + warp) * C::kWarpPartial;
                    };
                    float *part = part_of((int)blockIdx.x);
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld_32x32(to + 32 * c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            *reinterpret_cast<uint4 *>(part + ((8 * c + i) * 32 + lane) * 4) =
                                make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                    part[32 * D + lane] = m;
                    part[32 * D + 32 + lane] = l;
                    __threadfence();
                    __syncwarp();
                    int before = 0;
                    int *ticket = a.tickets + first * 8 + warp;
                    if (lane == 0) {
                        before = atomicAdd(ticket, 1);
                        if (before == final - first) *ticket = 0;  // zero again for the next launch
                    }
                    before = __shfl_sync(0xffffffffu, before, 0);
                    __threadfence();
                    if (before == final - first) {
                        float top = -INFINITY, sum = 0.0f;
                        for (int cta = first; cta <= final; ++cta) top = fmaxf(top, __ldcg(part_of(cta) + 32 * D + lane));
                        const float ref = top == -INFINITY ? 0.0f : top;
                        for (int cta = first; cta <= final; ++cta) {
                            const float *pc = part_of(cta) + 32 * D + lane;
                            sum = fmaf(__ldcg(pc + 32), fast_ex2((__ldcg(pc) - ref) * a.scale_log2), sum);
                        }
                        const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll 1
                        for (int c = 0; c < D / 8; ++c) {
                            float v[8] = {};
                            for (int cta = first; cta <= final; ++cta) {
                                const float *pc = part_of(cta);
                                const float f = fast_ex2((__ldcg(pc + 32 * D + lane) - ref) * a.scale_log2);
                                const float4 u0 = __ldcg(reinterpret_cast<const float4 *>(pc + ((2 * c) * 32 + lane) * 4));
                                const float4 u1 = __ldcg(reinterpret_cast<const float4 *>(pc + ((2 * c + 1) * 32 + lane) * 4));
                                v[0] = fmaf(u0.x, f, v[0]); v[1] = fmaf(u0.y, f, v[1]);
                                v[2] = fmaf(u0.z, f, v[2]); v[3] = fmaf(u0.w, f, v[3]);
                                v[4] = fmaf(u1.x, f, v[4]); v[5] = fmaf(u1.y, f, v[5]);
                                v[6] = fmaf(u1.z, f, v[6]); v[7] = fmaf(u1.w, f, v[7]);
                            }
                            if (live)
                                *reinterpret_cast<uint4 *>(dst + 8 * c) =
                                    make_uint4(Half2Of<T>::pack(v[0] * inv, v[1] * inv), Half2Of<T>::pack(v[2] * inv, v[3] * inv),
                                               Half2Of<T>::pack(v[4] * inv, v[5] * inv), Half2Of<T>::pack(v[6] * inv, v[7] * inv));
                        }
                    }
                }
                tc_fence_before_sync();  // O has been read before the next run's first product, which waits for p_ready
            }
            x = min(x1, end);
            if (x < x1) {
                __syncwarp();
                if (lane == 0) next_item<kChunkRows, kKeyTile>(a, it);
                __syncwarp();
            }
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag) {
        // a wait ran out: copies and products in flight get time to land before what they target is released
        const unsigned long long t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 200000ull) {
        }
        __syncthreads();
    }
    if (warp == 9) tmem_dealloc(tmem, 512);
}

typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                             const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_tiled() {
    static EncodeFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeFn>(p);
    });
    return fn;
}

// Pages as (64 elements of a head, tokens, heads, pages); a box is 64 elements of `page_box` tokens.
int make_page_map(CUtensorMap *map, void *base, const b200_w8a8_kv_cache *c, int page_box) {
    EncodeFn fn = encode_tiled();
    if (!fn) return fail("cuTensorMapEncodeTiled is not available from this driver");
    cuuint64_t dims[4] = {(cuuint64_t)c->d_head, (cuuint64_t)c->page_tokens, (cuuint64_t)c->n_kv_heads, (cuuint64_t)c->n_pages};
    cuuint64_t strides[3] = {(cuuint64_t)c->token_stride * 2, (cuuint64_t)c->head_stride * 2, (cuuint64_t)c->page_stride * 2};
    cuuint32_t box[4] = {64, (cuuint32_t)page_box, 1, 1}, one[4] = {1, 1, 1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, base, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail("paged_attention: these page strides cannot be described to the copy engine (%d)", (int)r);
    return 0;
}

template <typename T, int D>
int launch_chunk(const CUtensorMap &k, const CUtensorMap &v, const AttnParams &a, const ChunkExtra &ex, int sms, bool &attr_set,
                 cudaStream_t stream) {
    if (!attr_set) {
        cudaError_t e = cudaFuncSetAttribute(attention_chunk_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             ChunkCfg<D>::kSmemBytes);
        if (e != cudaSuccess) return fail("cudaFuncSetAttribute(attention_chunk): %s", cudaGetErrorString(e));
        attr_set = true;
    }
    launch_kernel(attention_chunk_kernel<T, D>, dim3(sms), dim3(kChunkThreads), ChunkCfg<D>::kSmemBytes, stream, k, v, a, ex);
    return check_launch("paged_attention (chunk)");
}

}  // namespace

size_t attention_chunk_partial_bytes(int d_head, int sms) { return (size_t)sms * 2 * 8 * 32 * (d_head + 2) * sizeof(float); }

int launch_attention_chunk(const b200_w8a8_kv_cache *cache, const AttnParams &a, int sms, int dev, cudaStream_t stream) {
    static bool attr_set[64][2][2];
    ChunkExtra ex{};
    ex.page_box = cache->page_tokens < kKeyTile ? cache->page_tokens : kKeyTile;
    ex.wait_limit_ns = wait_limit_ns();
    ex.debug_drop_load = take_debug_drop();
    CUtensorMap k, v;
    if (make_page_map(&k, cache->k_pages, cache, ex.page_box) || make_page_map(&v, cache->v_pages, cache, ex.page_box)) return 1;
    bool(&set)[2][2] = attr_set[dev & 63];
    const bool bf = cache->dtype == B200_DT_BF16;
    if (cache->d_head == 64)
        return bf ? launch_chunk<__nv_bfloat16, 64>(k, v, a, ex, sms, set[0][1], stream)
                  : launch_chunk<__half, 64>(k, v, a, ex, sms, set[0][0], stream);
    return bf ? launch_chunk<__nv_bfloat16, 128>(k, v, a, ex, sms, set[1][1], stream)
              : launch_chunk<__half, 128>(k, v, a, ex, sms, set[1][0], stream);
}

}  // namespace b200
