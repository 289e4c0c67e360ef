// Attention of many query rows per key head (chunks of prompts, frames): tcgen05 matrix products over KV tiles of 128 keys.
//
// A work item is 256 query rows of one (sequence, key head), as two tiles A and B of 128 rows.  Per KV tile and row tile
//     S = Q K^T (tensor memory, fp32)  ->  P = 2^(c (S - m)) (16 bits, over S in tensor memory)  ->  O += P V.
// One warp fetches pages by TMA into a ring of K and V tiles, one thread issues the products, and four warps each own the
// softmax of A and of B, one thread per row, so that row maxima and sums need no exchange.  While A's weights are computed the
// tensor core works on B.  The running maximum moves only when a row has outgrown it by 2^8 (weights stay below 2^8, and the
// factor cancels in the quotient), so O in tensor memory is rescaled rarely.  Weights are rounded to the cache's type, half a
// step each: that is what the tensor core takes; their sum is taken before, in fp32.  fp16 weights carry a factor 2^7 more, up to
// 2^15 in all, so that those of a long sequence beside a large one stay above the least number of that type (131071 keys
// beside one that is 2^26 times as large: without it their share of the output was lost).
// Keys stay K-major as they lie in the page, values are read in the same layout as the MN-major operand: nothing is
// transposed.  Rows of V outside the sequence are zeroed in shared memory before their product, since 0 x NaN is no zero.
// An item of at most 128 rows has no second row tile: both accumulators work on it, KV tiles in turn.
//
// Measured in a graph of a few passes: a prompt of 8192 tokens (32 / 8 heads of 128, bf16, causal) 475 us = 1.16 PFLOP/s, 70 % of
// the rate of a large library product; repeated without a pause it runs into the power cap, 545 us = 1.01 PFLOP/s.  A frame
// of 512 tokens over 8704 keys (32 / 16 heads of 64, fp16) 65 to 68 us, 80 rows of 16 sequences of up to 4001 keys (32 / 2 heads of
// 128) 28 us.  In the prompt the tensor pipe is busy 60 % of the
// cycles, the special-function unit 45 %, the issue slots 46 %: what bounds the loop is the chain scores -> maximum -> weights
// -> product of a row tile (about 3400 cycles a KV tile, of which the products are 1000), of which two run against each other.
// Tried and slower: half a row per thread with sixteen softmax warps (563 us), KV tiles in halves with two score buffers (517),
// a thread per row tile to issue products (583 when their batches mix, 501 when the softmax warps take turns), all
// exponentials on the special-function unit (476), rolled loops over 32 scores (529).
#include <cuda.h>

#include <algorithm>
#include <mutex>

#include "paged_attention.cuh"

namespace b200 {
namespace {

constexpr int kChunkThreads = 384;  // three warpgroups; warps 10 and 11 only fill the third
// registers a thread: 384 x 168 at launch = 64512 = 256 x 224 + 128 x 56
constexpr int kSoftmaxRegs = 224, kOtherRegs = 56;
constexpr int kSlabBytes = 128 * 128;  // 128 rows of 64 16-bit elements, 128-byte swizzle
constexpr float kLazyRescale = 8.0f;   // log2 of how far a weight may exceed one
constexpr float kWeightsUp = 7.0f;     // log2 of the factor of fp16 weights
constexpr int kJoinAtOnce = 8;         // parts of an item that are joined in one step; 32 rows over 60000 keys, all at once 101 us, so 37

template <int D>
struct ChunkCfg {
    static constexpr int kTileBytes = D / 64 * kSlabBytes;
    static constexpr int kStages = D == 128 ? 5 : 8;
    static constexpr int kBars = 2 * kStages + 18;
    static constexpr int kSmemBytes = (2 + kStages) * kTileBytes + kBars * 8 + 16 + 1024;  // and alignment
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
// True in one thread of a converged warp.  Unlike `lane == 0` the compiler knows that a branch on it holds a single thread, and
// feeds the operands of tcgen05 instructions to the uniform registers directly.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(one));
    return one != 0;
}
// Four products over 16 elements of K each: 32 bytes of a K-major row, or 8 columns of weights and 16 rows of values.  One block
// of assembly with its own arithmetic: left to the compiler, the operands of all unrolled products are kept in registers that the
// issuing warp does not have.
__device__ __forceinline__ void umma_f16_ss4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, t;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "add.s64 a, %1, 2;\n\tadd.s64 b, %2, 2;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t"
        "add.s64 a, %1, 4;\n\tadd.s64 b, %2, 4;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t"
        "add.s64 a, %1, 6;\n\tadd.s64 b, %2, 6;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void umma_f16_ts4(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, t;\n\t.reg .b32 a;\n\t.reg .b64 b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "add.u32 a, %1, 8;\n\tadd.s64 b, %2, 128;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "add.u32 a, %1, 16;\n\tadd.s64 b, %2, 256;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "add.u32 a, %1, 24;\n\tadd.s64 b, %2, 384;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t}" ::"r"(d),
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
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
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

// 2^x for x in [-inf, 127] on the multiply-add pipe: x = n + f, n the nearest integer, |f| <= 1/2; 2^f by the polynomial of
// least relative error over that interval among those that are exact at 0 (degree 3: 1.0e-4, for weights rounded to bf16 by
// up to 2^-9; degree 4: 2.8e-6, for fp16's 2^-12), times 2^n.  x <= -126.5, -inf too, gives exactly 0, NaN gives NaN: n added
// to the exponent as an integer would be a step less, and make a large finite number of it.
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
template <int DEGREE>
__device__ __forceinline__ void poly_ex2(uint64_t x, float &e0, float &e1) {
    float a, b;
    unpair2(x, a, b);
    x = pair2(max_nan(a, -127.0f), max_nan(b, -127.0f));
    // 1.5 * 2^23 + 127: adding it rounds to an integer, and leaves n + 127, the exponent of 2^n, in the low bits
    const float magic = 12583039.0f;
    const uint64_t one = pair2(1.0f, 1.0f), t = add2(x, pair2(magic, magic));
    const uint64_t f = fma2(add2(t, pair2(-magic, -magic)), pair2(-1.0f, -1.0f), x);
    uint64_t p;
    if (DEGREE == 3) {
        p = fma2(pair2(0.05500893294811249f, 0.05500893294811249f), f, pair2(0.2422109693288803f, 0.2422109693288803f));
        p = fma2(p, f, pair2(0.6932829022407532f, 0.6932829022407532f));
    } else {
        p = fma2(pair2(0.009585382416844368f, 0.009585382416844368f), f, pair2(0.05590662732720375f, 0.05590662732720375f));
        p = fma2(p, f, pair2(0.24024038016796112f, 0.24024038016796112f));
        p = fma2(p, f, pair2(0.6931241750717163f, 0.6931241750717163f));
    }
    p = fma2(p, f, one);
    float t0, t1;
    unpair2(t, t0, t1);
    unpair2(mul2(p, pair2(__int_as_float(__float_as_int(t0) << 23), __int_as_float(__float_as_int(t1) << 23))), e0, e1);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
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

// Of every 8 pairs of weights, how many the multiply-add pipe computes.  Measured, 1 / 2 / 3 / 4 / 5 of 8: a frame of 512 tokens
// over 8704 keys, d = 64: 66.3 / - / 63.5 / 68.3 / 73.1 us; a prompt of 8192 tokens, d = 128: 476 / 470 / 480 / 523 / 530 us.
template <int D>
constexpr int kPolyPairs = D == 128 ? 2 : 3;

// Waits and commits by shared-memory address: what stands between two products of the issuing thread is kept short.
constexpr uint32_t kWaitNs = 20000;  // how long one try of a wait may sleep; measured, it sleeps about 4 us
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "n"(kWaitNs)
        : "memory");
    return ok != 0;
}
// Waits with a limit, in units of 1024 ns; false when it runs out or another warp's has: *abort then holds the first code, which
// is reported when the CTA ends.  The clock is read after a first try.  Measured against a look at it every 64 tries: frame 67.1
// against 69.6 us, prompt 473 against 483 us.
__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity, volatile int *abort, unsigned limit, int code) {
    if (try_wait(bar, parity)) return true;
    const unsigned begin = (unsigned)(global_timer_ns() >> 10);
#pragma unroll 1
    while (!try_wait(bar, parity)) {
        if (*abort) return false;
        if ((unsigned)(global_timer_ns() >> 10) - begin > limit) {
            *abort = code;
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ void commit_to(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_on(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

struct ChunkExtra {
    int page_box;  // tokens per TMA box: min(page_tokens, 128)
    unsigned wait_limit;  // of one wait, in units of 1024 ns
    int debug_drop_load;
};

// An item of one row tile: both accumulators work on it, KV tiles in turn, and are joined at the end of a run.  Of other items
// both row tiles hold rows.
__device__ __forceinline__ bool is_shared(const Item &it) { return it.rows - it.rt * kChunkRows <= 128; }

template <typename T, int D>
__global__ void __launch_bounds__(kChunkThreads, 1)
    attention_chunk_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                           const AttnParams a, const ChunkExtra ex) {
    using C = ChunkCfg<D>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ PlanShared<kChunkThreads> plan;
    __shared__ Walk walks[10];  // every warp's own, kept out of the loops' registers
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *ring = smem + 2 * C::kTileBytes;
    // barriers: [stage] pages have landed; [stage] their products are done; [row tile] its queries are in shared memory; its
    // scores are in tensor memory; [row tile][half] half of its weights are there and O is rescaled; [row tile] the last product
    // of a run has landed; [warp] where both work on one row tile: B's maxima and sums are known, and A has taken B's part over
    uint64_t *bars = reinterpret_cast<uint64_t *>(ring + C::kStages * C::kTileBytes);
    const uint32_t kv_full = smem_u32(bars), kv_empty = kv_full + 8 * C::kStages, q_ready = kv_empty + 8 * C::kStages;
    const uint32_t s_full = q_ready + 16, p_ready = s_full + 16, o_full = p_ready + 32;
    const uint32_t b_known = o_full + 16, b_taken = b_known + 32;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + C::kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    pdl_trigger();
    if (threadIdx.x == 0) {
        // four arrivals, one per softmax warp, where such a warp signals; one everywhere else
        for (int i = 0; i < C::kBars; ++i) {
            const int j = i - 2 * C::kStages;
            mbar_init(bars + i, j == 0 || j == 1 || (j >= 4 && j < 8) ? 4 : 1);
        }
        *abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
    }
    pdl_wait();
    {
        Walk w;
        if (!plan_run<kChunkRows, kKeyTile, kChunkExtra, kChunkThreads>(a, plan, w.map, w.x, w.x1, w.it)) return;
        w.locate<kChunkExtra>();
        if (lane == 0 && warp < 10) walks[warp] = w;
    }
    Walk &walk = walks[min(warp, 9)];
    const volatile Walk &now = walk;
    Item &it = walk.it;
    // one lane takes the warp's walk to its next item
    auto advance = [&]() {
        __syncwarp();
        if (lane == 0) walk.advance<kChunkRows, kKeyTile, kChunkExtra>(a);
        __syncwarp();
    };
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
            while (ok && now.kt0 < now.kt1) {
                const int kt0 = now.kt0, kt1 = now.kt1;
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
                        ok = wait_bounded(kv_empty + 8 * s, ph ^ 1u, abort_flag, ex.wait_limit, KS_TIMEOUT_SMEM_EMPTY);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(bars + s, bytes);
                        __syncwarp();
                        if (live && !drop) {
                            const uint32_t dst = smem_u32(ring + s * C::kTileBytes) + (uint32_t)(lane * ex.page_box * 128);
#pragma unroll
                            for (int d = 0; d < D / 64; ++d)
                                tma_load_4d(dst + d * kSlabBytes, kv ? &tm_v : &tm_k, bars + s, d * 64, token, kv_head, page);
                        }
                        drop = false;
                        if (++s == C::kStages) { s = 0; ph ^= 1u; }
                    }
                }
                advance();
            }
        } else if (warp == 9) {
            // ---- products, all issued by one thread
            if (elect_one()) {
                constexpr uint32_t idesc_s = idesc_f16<T>(kKeyTile, 0), idesc_o = idesc_f16<T>(D, 1);
                const uint64_t q_desc = umma_smem_desc_k128(smem_u32(smem)), k_desc = umma_smem_desc_k128(smem_u32(ring));
                const uint64_t v_desc = smem_desc_mn128(smem_u32(ring));
                int s = 0;
                uint32_t ph = 0, q_ph = 0, p_ph = 0;  // q_ph, p_ph: bit x is the parity of row tile x's barriers
                while (now.kt0 < now.kt1) {
                    const int kt0 = now.kt0, kt1 = now.kt1;
                    bool ok = true;
                    if (is_shared(it)) {
                        // one row tile, whose queries serve both accumulators: A takes the run's KV tiles 0, 2, ..., B 1, 3, ...
                        const int n = kt1 - kt0;
                        auto ahead = [&](int by, uint32_t &bar, uint32_t &par) {  // stage `by` behind s, its barrier and parity
                            int st = s + by;
                            par = ph;
                            if (st >= C::kStages) { st -= C::kStages; par ^= 1u; }
                            bar = kv_full + 8 * st;
                            return st;
                        };
                        ok = wait_bounded(q_ready, q_ph & 1u, abort_flag, ex.wait_limit, KS_TIMEOUT_SOFTMAX);
                        q_ph ^= 1u;
                        tc_fence_after_sync();
#pragma unroll 1
                        for (int i = -2; ok && i < n; ++i) {
                            const int r = i & 1;
                            uint32_t bar, par;
                            if (i >= 0) {
                                const int vs = ahead(1, bar, par);
                                ok = wait_bounded(bar, par, abort_flag, ex.wait_limit, KS_TIMEOUT_SMEM_FULL);
                                const uint64_t vd = v_desc + (uint64_t)(vs * (C::kTileBytes >> 4));
#pragma unroll 1
                                for (int half = 0; ok && half < 2; ++half) {
                                    ok = wait_bounded(p_ready + 16 * r + 8 * half, (p_ph >> r) & 1u, abort_flag, ex.wait_limit,
                                                      KS_TIMEOUT_SOFTMAX);
                                    if (!ok) break;
                                    tc_fence_after_sync();
                                    umma_f16_ts4(tmem_o + r * D, tmem + r * kKeyTile + 32 * half,
                                                 vd + (uint64_t)(half * (64 * 128 >> 4)), idesc_o, i >= 2 || half);
                                }
                                if (!ok) break;
                                p_ph ^= 1u << r;
                                if (i + 2 >= n) commit_to(o_full + 8 * r);
                                commit_to(kv_empty + 8 * vs);
                            }
                            if (i + 2 < n) {  // K of tile i + 2: its stage is two for each tile ahead of tile max(i, 0)'s
                                const int ks = ahead(2 * (i + 2 - (i > 0 ? i : 0)), bar, par);
                                ok = wait_bounded(bar, par, abort_flag, ex.wait_limit, KS_TIMEOUT_SMEM_FULL);
                                if (!ok) break;
                                tc_fence_after_sync();
                                const uint64_t kd = k_desc + (uint64_t)(ks * (C::kTileBytes >> 4));
#pragma unroll
                                for (int d = 0; d < D / 64; ++d)
                                    umma_f16_ss4(tmem + r * kKeyTile, q_desc + (uint64_t)(d * (kSlabBytes >> 4)),
                                                 kd + (uint64_t)(d * (kSlabBytes >> 4)), idesc_s, d != 0);
                                commit_to(s_full + 8 * r);
                                commit_to(kv_empty + 8 * ks);
                            }
                            if (i >= 0) {
                                s += 2;
                                if (s >= C::kStages) { s -= C::kStages; ph ^= 1u; }
                            }
                        }
                        if (!ok) break;
                        walk.advance<kChunkRows, kKeyTile, kChunkExtra>(a);
                        continue;
                    }
                    for (int kt = kt0 - 1; kt < kt1; ++kt) {
                        // V of tile kt and K of tile kt + 1 are the next two stages of the ring
                        const int vs = s;
                        if (kt >= kt0) {
                            ok = wait_bounded(kv_full + 8 * s, ph, abort_flag, ex.wait_limit, KS_TIMEOUT_SMEM_FULL);
                            if (++s == C::kStages) { s = 0; ph ^= 1u; }
                        }
                        const int ks = s;
                        if (kt + 1 < kt1 && ok) {
                            ok = wait_bounded(kv_full + 8 * s, ph, abort_flag, ex.wait_limit, KS_TIMEOUT_SMEM_FULL);
                            if (++s == C::kStages) { s = 0; ph ^= 1u; }
                        }
                        if (!ok) break;
#pragma unroll 1
                        for (int r = 0; r < 2; ++r) {
                            if (kt >= kt0) {
                                const uint64_t vd = v_desc + (uint64_t)(vs * (C::kTileBytes >> 4));
                                const uint32_t par = (p_ph >> r) & 1u;
#pragma unroll 1
                                for (int half = 0; half < 2; ++half) {
                                    ok = wait_bounded(p_ready + 16 * r + 8 * half, par, abort_flag, ex.wait_limit, KS_TIMEOUT_SOFTMAX);
                                    if (!ok) break;
                                    tc_fence_after_sync();
                                    umma_f16_ts4(tmem_o + r * D, tmem + r * kKeyTile + 32 * half,
                                                 vd + (uint64_t)(half * (64 * 128 >> 4)), idesc_o, kt != kt0 || half);
                                }
                                if (!ok) break;
                                p_ph ^= 1u << r;
                                if (kt + 1 == kt1) commit_to(o_full + 8 * r);
                            } else {
                                ok = wait_bounded(q_ready + 8 * r, (q_ph >> r) & 1u, abort_flag, ex.wait_limit, KS_TIMEOUT_SOFTMAX);
                                if (!ok) break;
                                q_ph ^= 1u << r;
                                tc_fence_after_sync();
                            }
                            // the products of one CTA execute in the order of their issue, so scores are written over weights
                            // only after the product that reads these
                            if (kt + 1 < kt1) {
                                const uint64_t qd = q_desc + (uint64_t)(r * (C::kTileBytes >> 4));
                                const uint64_t kd = k_desc + (uint64_t)(ks * (C::kTileBytes >> 4));
#pragma unroll
                                for (int d = 0; d < D / 64; ++d)
                                    umma_f16_ss4(tmem + r * kKeyTile, qd + (uint64_t)(d * (kSlabBytes >> 4)),
                                                 kd + (uint64_t)(d * (kSlabBytes >> 4)), idesc_s, d != 0);
                                commit_to(s_full + 8 * r);
                            }
                        }
                        if (!ok) break;
                        if (kt >= kt0) commit_to(kv_empty + 8 * vs);
                        if (kt + 1 < kt1) commit_to(kv_empty + 8 * ks);
                    }
                    if (!ok) break;
                    walk.advance<kChunkRows, kKeyTile, kChunkExtra>(a);
                }
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        // ---- softmax: warps 0-3 own row tile A, 4-7 row tile B; a thread owns a row
        const int tile = warp >> 2, sub = warp & 3;
        const uint32_t lanes = (uint32_t)(sub * 32) << 16;
        const uint32_t ts = tmem + lanes + tile * kKeyTile, to = tmem_o + lanes + tile * D;
        constexpr int kChunks = D / 8;          // 16-byte chunks of a row
        constexpr int kRowsPerPass = 32 / kChunks;
        // The warp's 32 rows of shared memory: queries in the swizzled K-major layout, and after a run the way of its results
        // to memory.  Global memory is accessed kRowsPerPass whole rows at a time.
        uint8_t *mine = smem + tile * C::kTileBytes + sub * 32 * 128;
        auto chunk_at = [&](int row, int c) { return mine + (c / 8) * kSlabBytes + row * 128 + (((c & 7) ^ (row & 7)) << 4); };
        const int pass_row = lane / kChunks, pass_chunk = lane % kChunks;
        auto q_at = [&](int r) {
            const int tok = a.by_group.div(r), head = it.h * a.group + r - tok * a.group;
            return reinterpret_cast<const T *>(a.q) + (it.seq.q0 + tok) * a.q_ts + head * a.q_hs + pass_chunk * 8;
        };
        auto load_q = [&](int row0) {
            uint4 qv[kChunks];
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                const int r = row0 + i * kRowsPerPass + pass_row;
                qv[i] = make_uint4(0, 0, 0, 0);
                if (r < it.rows) qv[i] = *reinterpret_cast<const uint4 *>(q_at(r));
            }
#pragma unroll
            for (int i = 0; i < kChunks; ++i)
                *reinterpret_cast<uint4 *>(chunk_at(i * kRowsPerPass + pass_row, pass_chunk)) = qv[i];
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) arrive_on(q_ready + 8 * tile);
        };
        uint32_t s_ph = 0, o_ph = 0, b_ph = 0, known_ph = 0;  // b_ph: of B's o_full, as A sees it
        const float *b_stats = reinterpret_cast<const float *>(smem + C::kTileBytes + sub * 32 * 128);  // in B's idle queries
        int tiles_before = 0;  // KV tiles of this CTA before the current run: where in the ring its values arrive
        bool ok = true, first_run = true;
        while (now.kt0 < now.kt1) {
            const int kt0 = now.kt0, kt1 = now.kt1;
            const bool shared = is_shared(it);
            const int row0 = it.rt * kChunkRows + (shared ? 0 : tile * 128) + sub * 32;
            const int kt_first = shared ? kt0 + tile : kt0, kt_step = shared ? 2 : 1;
            float m = -INFINITY, l = 0.0f;
            const int item_lo = it.lo, item_hi = it.hi;
            if (first_run && (tile == 0 || !shared)) load_q(row0);
            int lo = 0, hi = 0x7fffffff;  // a row that is not there masks nothing
            if (row0 + lane < it.rows)
                visible_keys(a, it.seq.keys - it.seq.n + a.by_group.div(row0 + lane), it.seq.keys, lo, hi);
            const int lo_max = __reduce_max_sync(0xffffffffu, lo), hi_min = __reduce_min_sync(0xffffffffu, hi);
            for (int kt = kt_first; kt < kt1; kt += kt_step) {
                ok = wait_bounded(s_full + 8 * tile, s_ph, abort_flag, ex.wait_limit, KS_TIMEOUT_SOFTMAX);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                s_ph ^= 1u;
                tc_fence_after_sync();
                // Values of keys that the item's rows do not see may be anything, NaN too, and 0 x NaN is no zero: the four
                // warps whose product comes first clear them before their weights let it begin
                if ((tile == 0 || shared) && (kt * kKeyTile < item_lo || (kt + 1) * kKeyTile > item_hi)) {
                    const unsigned at = 2u * (unsigned)(tiles_before + kt - kt0) + 1u, stage = at % C::kStages;
                    ok = __all_sync(0xffffffffu, wait_bounded(kv_full + 8 * stage, at / C::kStages & 1u, abort_flag,
                                                              ex.wait_limit, KS_TIMEOUT_SMEM_FULL));
                    if (!ok) break;
                    uint8_t *v = ring + stage * C::kTileBytes;
                    for (int row = sub * 32 + lane / 8; row < sub * 32 + 32; row += 4) {
                        const int key = kt * kKeyTile + row;
                        if (key < item_lo || key >= item_hi) {
#pragma unroll
                            for (int d = 0; d < D / 64; ++d)
                                *reinterpret_cast<uint4 *>(v + d * kSlabBytes + row * 128 + (lane & 7) * 16) =
                                    make_uint4(0, 0, 0, 0);
                        }
                    }
                    fence_proxy_async_smem();
                }
                uint32_t s[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld_32x32(ts + 32 * c, s[c]);
                tmem_ld_wait();
                auto f = [&](int i) { return __uint_as_float(s[i / 32][i % 32]); };
                const int key0 = kt * kKeyTile;
                if (key0 < lo_max || key0 + kKeyTile > hi_min) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int from = lo - key0 - 32 * c, upto = hi - key0 - 32 * c;
                        if (lo_max > key0 + 32 * c) {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (i < from) s[c][i] = 0xff800000u;
                        }
                        if (hi_min < key0 + 32 * c + 32) {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (i >= upto) s[c][i] = 0xff800000u;
                        }
                    }
                }
                float t8[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    t8[i] = f(i);
#pragma unroll
                    for (int j = 8; j < kKeyTile - 8; j += 16) t8[i] = max3(t8[i], f(i + j), f(i + j + 8));
                    t8[i] = fmaxf(t8[i], f(i + kKeyTile - 8));
                }
                const float top = max3(max3(t8[0], t8[1], t8[2]), max3(t8[3], t8[4], t8[5]), fmaxf(t8[6], t8[7]));
                if (kt == kt_first) {
                    m = top;
                } else if (__any_sync(0xffffffffu, (top - m) * a.scale_log2 > kLazyRescale)) {
                    const float mn = fmaxf(m, top);
                    const float g = m == -INFINITY ? 0.0f : fast_ex2((m - mn) * a.scale_log2);
                    m = mn;
                    l *= g;
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t o[16];
                        tmem_ld_32x16(to + 16 * c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * g);
                        tmem_st_32x16(to + 16 * c, o);
                    }
                }
                const float ref = m == -INFINITY ? 0.0f : m * a.scale_log2 - (IsBf16<T>::value ? 0.0f : kWeightsUp);
                const uint64_t scale2 = pair2(a.scale_log2, a.scale_log2), ref2 = pair2(-ref, -ref);
                uint64_t sum[4] = {};
                // weights of 32 keys at a time over the scores, which are in registers by now.  Some pairs go to the
                // multiply-add pipe, the others to the special-function unit, which alone would bound the kernel.
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const uint64_t v = fma2(pair2(f(32 * c + 2 * i), f(32 * c + 2 * i + 1)), scale2, ref2);
                        float e0, e1;
                        if ((i & 7) < kPolyPairs<D>) {
                            poly_ex2<IsBf16<T>::value ? 3 : 4>(v, e0, e1);
                        } else {
                            unpair2(v, e0, e1);
                            e0 = fast_ex2(e0);
                            e1 = fast_ex2(e1);
                        }
                        sum[i & 3] = add2(sum[i & 3], pair2(e0, e1));
                        w[i] = Half2Of<T>::pack(e0, e1);
                    }
                    tmem_st_32x16(ts + 16 * c, w);
                    if (c & 1) {  // half of the weights: their product may begin
                        tmem_st_wait();
                        tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) arrive_on(p_ready + 16 * tile + 8 * (c / 2));
                    }
                }
                float l0, l1;
                unpair2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), l0, l1);
                l += l0 + l1;
            }
            if (!ok) break;
            // what the end of this run needs, then on to the next item, whose queries come to L2 meanwhile
            tiles_before += kt1 - kt0;
            const int first = now.first, final = now.final, rows = it.rows, head0 = it.h * a.group, q0 = it.seq.q0;
            advance();
            const bool more = now.kt0 < now.kt1 && it.rt * kChunkRows + tile * 128 < it.rows;  // queries to fetch
            {
                const int r = it.rt * kChunkRows + tile * 128 + sub * 32 + lane;
                if (more && r < it.rows) {
#pragma unroll
                    for (int d = 0; d < D; d += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(q_at(r) - pass_chunk * 8 + d));
                }
            }
            first_run = false;
            const bool mine_any = kt_first < kt1;  // B has nothing in a run of one KV tile
            if (shared && tile == 1) {
                float *stats = const_cast<float *>(b_stats);
                stats[lane] = m;
                stats[32 + lane] = l;
                __syncwarp();
                if (lane == 0) arrive_on(b_known + 8 * sub);
                ok = wait_bounded(b_taken + 8 * sub, known_ph, abort_flag, ex.wait_limit, KS_TIMEOUT_TMEM_FULL);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                known_ph ^= 1u;
                if (mine_any) o_ph ^= 1u;
                if (more) load_q(it.rt * kChunkRows + tile * 128 + sub * 32);
                continue;
            }
            ok = wait_bounded(o_full + 8 * tile, o_ph, abort_flag, ex.wait_limit, KS_TIMEOUT_TMEM_FULL);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            o_ph ^= 1u;
            // this row's factors of the two accumulators
            float fa = 1.0f, fb = 0.0f;
            if (shared) {
                const bool b_any = kt0 + 1 < kt1;
                ok = wait_bounded(b_known + 8 * sub, known_ph, abort_flag, ex.wait_limit, KS_TIMEOUT_TMEM_FULL);
                if (ok && b_any) ok = wait_bounded(o_full + 8, b_ph, abort_flag, ex.wait_limit, KS_TIMEOUT_TMEM_FULL);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                known_ph ^= 1u;
                if (b_any) {
                    b_ph ^= 1u;
                    const float mb = b_stats[lane], lb = b_stats[32 + lane], top = fmaxf(m, mb);
                    const float ref = top == -INFINITY ? 0.0f : top;
                    fa = fast_ex2((m - ref) * a.scale_log2);
                    fb = fast_ex2((mb - ref) * a.scale_log2);
                    m = top;
                    l = l * fa + lb * fb;
                }
            } else {
                b_ph ^= 1u;
            }
            const bool two = shared && kt0 + 1 < kt1;
            auto b_done = [&]() {  // B may go on to its next run
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) arrive_on(b_taken + 8 * sub);
            };
            auto load_o = [&](int c, float (&o)[32]) {  // columns 32 c .. of this row's sum
                uint32_t u[32];
                tmem_ld_32x32(to + 32 * c, u);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(u[i]);
                if (two) {
                    tmem_ld_32x32(to + D + 32 * c, u);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = fmaf(__uint_as_float(u[i]), fb, o[i] * fa);
                }
            };
            tc_fence_after_sync();
            bool write = first == final;
            if (row0 >= rows) {  // none of the warp's rows is there
                write = false;
                if (shared) b_done();
            } else if (write) {
                const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    float o[32];
                    load_o(c, o);
                    auto g = [&](int i) { return o[i] * inv; };
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<uint4 *>(chunk_at(lane, 4 * c + i)) =
                            make_uint4(Half2Of<T>::pack(g(8 * i), g(8 * i + 1)), Half2Of<T>::pack(g(8 * i + 2), g(8 * i + 3)),
                                       Half2Of<T>::pack(g(8 * i + 4), g(8 * i + 5)), Half2Of<T>::pack(g(8 * i + 6), g(8 * i + 7)));
                }
                if (shared) b_done();
            } else {
                // [slot of the CTA][warp]: columns in vectors of four, 32 rows each
                const int parts = final - first + 1;
                auto slot_of = [&](int cta) {
                    return a.partials + ((long long)(2 * cta + (cta == first ? 1 : 0)) * 8 + warp) * C::kWarpPartial;
                };
                float *part = slot_of((int)blockIdx.x);
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    float o[32];
                    load_o(c, o);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *reinterpret_cast<float4 *>(part + ((8 * c + i) * 32 + lane) * 4) =
                            make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                }
                if (shared) b_done();
                part[32 * D + lane] = m;
                part[32 * D + 32 + lane] = l;
                // whether this warp is the last of n to arrive at a counter; then the others' parts can be read
                auto last_of = [&](int *ticket, int n) {
                    __threadfence();
                    __syncwarp();
                    int before = 0;
                    if (lane == 0) {
                        before = atomicAdd(ticket, 1);
                        if (before == n - 1) *ticket = 0;  // zero again for the next launch
                    }
                    before = __shfl_sync(0xffffffffu, before, 0);
                    __threadfence();
                    return before == n - 1;
                };
                // joins parts of the CTAs from, from + step, ...: maximum and sum, then 32 columns at a time to `sink`
                auto join = [&](int from, int step, int n, float &top, float &sum, auto &&sink) {
                    top = -INFINITY;
                    sum = 0.0f;
                    for (int h = 0; h < n; h += 8) {  // eight loads on the way; behind the last part, it once more
                        float m8[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) m8[i] = __ldcg(slot_of(from + min(h + i, n - 1) * step) + 32 * D + lane);
#pragma unroll
                        for (int i = 0; i < 8; ++i) top = fmaxf(top, m8[i]);
                    }
                    const float ref = top == -INFINITY ? 0.0f : top;
                    for (int h = 0; h < n; h += 8) {
                        float m8[8], l8[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float *pc = slot_of(from + min(h + i, n - 1) * step) + 32 * D + lane;
                            m8[i] = __ldcg(pc);
                            l8[i] = __ldcg(pc + 32);
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (h + i < n) sum = fmaf(l8[i], fast_ex2((m8[i] - ref) * a.scale_log2), sum);
                    }
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        float v[32] = {};
#pragma unroll 3
                        for (int i = 0; i < n; ++i) {
                            const float *pc = slot_of(from + i * step);
                            const float g = fast_ex2((__ldcg(pc + 32 * D + lane) - ref) * a.scale_log2);
                            float4 u[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) u[j] = __ldcg(reinterpret_cast<const float4 *>(pc) + (8 * c + j) * 32 + lane);
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                v[4 * j] = fmaf(u[j].x, g, v[4 * j]);
                                v[4 * j + 1] = fmaf(u[j].y, g, v[4 * j + 1]);
                                v[4 * j + 2] = fmaf(u[j].z, g, v[4 * j + 2]);
                                v[4 * j + 3] = fmaf(u[j].w, g, v[4 * j + 3]);
                            }
                        }
                        sink(c, v);
                    }
                };
                // Many parts are joined in two steps, groups first, since one warp reads a part in more than a microsecond.  A
                // CTA begins at most one shared item and continues at most one, so a counter per CTA, warp and use is enough.
                int span = 1, n = parts;
                bool go = true;
                if (parts > kJoinAtOnce) {
                    span = (int)ceilf(sqrtf((float)parts));
                    n = (parts + span - 1) / span;
                    const int group = ((int)blockIdx.x - first) / span, from = first + group * span;
                    const int members = min(span, final - from + 1);
                    go = last_of(a.tickets + (from * 3 + (group == 0 ? 1 : 2)) * 8 + warp, members);
                    if (go) {  // the group's parts become one, in the place of its first
                        float top, sum;
                        float *to_slot = slot_of(from);
                        join(from, 1, members, top, sum, [&](int c, float(&v)[32]) {
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                *(reinterpret_cast<float4 *>(to_slot) + (8 * c + j) * 32 + lane) =
                                    make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                        });
                        to_slot[32 * D + lane] = top;
                        to_slot[32 * D + 32 + lane] = sum;
                    }
                }
                if (go && last_of(a.tickets + first * 3 * 8 + warp, n)) {
                    // the last for these rows joins what there is, in the order of its keys
                    write = true;
                    float top, sum;
                    join(first, span, n, top, sum, [&](int c, float(&v)[32]) {
                        const float w = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            *reinterpret_cast<uint4 *>(chunk_at(lane, 4 * c + i)) =
                                make_uint4(Half2Of<T>::pack(v[8 * i] * w, v[8 * i + 1] * w),
                                           Half2Of<T>::pack(v[8 * i + 2] * w, v[8 * i + 3] * w),
                                           Half2Of<T>::pack(v[8 * i + 4] * w, v[8 * i + 5] * w),
                                           Half2Of<T>::pack(v[8 * i + 6] * w, v[8 * i + 7] * w));
                    });
                }
            }
            if (write) {
                __syncwarp();
#pragma unroll
                for (int i = 0; i < kChunks; ++i) {
                    const int row = i * kRowsPerPass + pass_row, r = row0 + row;
                    const uint4 v = *reinterpret_cast<const uint4 *>(chunk_at(row, pass_chunk));
                    if (r < rows) {
                        const int tok = a.by_group.div(r), head = head0 + r - tok * a.group;
                        *reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.out) + (q0 + tok) * a.o_ts + head * a.o_hs +
                                                   pass_chunk * 8) = v;
                    }
                }
                __syncwarp();
            }
            tc_fence_before_sync();  // O has been read before the next run's first product, which waits for p_ready
            if (more) load_q(it.rt * kChunkRows + tile * 128 + sub * 32);
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag) {
        if (threadIdx.x == 0 && a.c.status && *(volatile int *)a.c.status == 0) {
            *(volatile int *)a.c.status = *abort_flag;
            __threadfence_system();
        }
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
    if (raise_smem_limit(attr_set, attention_chunk_kernel<T, D>, ChunkCfg<D>::kSmemBytes, "attention_chunk")) return 1;
    launch_kernel(attention_chunk_kernel<T, D>, dim3(sms), dim3(kChunkThreads), ChunkCfg<D>::kSmemBytes, stream, k, v, a, ex);
    return check_launch("paged_attention (chunk)");
}

}  // namespace

size_t attention_chunk_partial_bytes(int d_head, int sms) { return (size_t)sms * 2 * 8 * 32 * (d_head + 2) * sizeof(float); }

int launch_attention_chunk(const b200_w8a8_kv_cache *cache, const AttnParams &a, int sms, int dev, cudaStream_t stream) {
    static bool attr_set[64][2][2];
    ChunkExtra ex{};
    ex.page_box = cache->page_tokens < kKeyTile ? cache->page_tokens : kKeyTile;
    ex.wait_limit = (unsigned)std::min(wait_limit_ns() / 1024 + 1, 1ull << 30);
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
