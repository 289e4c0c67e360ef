// Attention of new tokens over the paged cache: host entry, and the kernel for few query rows per key head (decoding,
// drafts).  o = sum_j 2^(c (s_j - m)) v_j / sum_j 2^(c (s_j - m)) with s_j = q . k_j, c = scale * log2(e), in one pass over
// the keys with a running maximum m: when a step raises m, what has been summed so far is multiplied by 2^(c (m_old - m)).
// The reference's attention over its ring is src/world_cuda.cu:1960-2056.
//
// Few rows per key mean every key and value is used once or a few times: HBM bounds the kernel.  So its shape serves the
// loads: each warp streams its own 16 keys per step through a private ring of cp.async stages (no barrier of the CTA in the
// loop), 192 KB per SM in all, while 16-row matrix instructions, of which decoding uses as few as one row, do the arithmetic
// in a fraction of the loads' time.  A step's keys lie in one page (pages hold a multiple of 16 tokens).  A result and the
// weights are rounded once each to the cache's type; scores, maxima, sums and O are fp32.
//
// Measured: 64 sequences of up to 8191 keys (32 / 8 heads of 128, bf16) 246 us = 6.5 TB/s, what a plain copy reaches; one of
// 131071 keys 95 us = 5.7 TB/s (of the rest about 5 us are launch, plan and first loads, 4 us the join); one of 777 keys
// (32 / 16 heads of 64) 10 us, all latency: plan, first loads, parts and join, each behind the one before.
#include <algorithm>
#include <mutex>

#include "paged_attention.cuh"

namespace b200 {
namespace {

constexpr int kRowsThreads = 128;
constexpr int kRowTile = 16;  // rows of one matrix instruction
constexpr int kStepKeys = 16;
constexpr int kRowsKeyTile = kStepKeys * (kRowsThreads / 32);  // keys per KV tile of the plan
// measured 0 / 2 / 5: one sequence of 777 keys 12.7 / 11.2 / 10.3 us (more units, so more parts, which min_tiles below gives it
// as well), one of 131071 keys 95.8 / 94.0 / 93.3 us
constexpr int kRowsExtra = 2;

// log2 of a factor that all weights carry, and that cancels: the largest is 2^15 in fp16, whose least normal number is 2^-14, so
// that the many small weights of a long sequence beside a large one are not lost.
template <typename T>
constexpr float kWeightsUp = 0.0f;
template <>
constexpr float kWeightsUp<__half> = 15.0f;

template <int D>
struct RowsCfg {
    static constexpr int kStepBytes = 2 * kStepKeys * D * 2;  // keys and values of a step
    static constexpr int kStages = D == 128 ? 3 : 6;
    static constexpr int kSmemBytes = (kRowsThreads / 32) * kStages * kStepBytes;
    static constexpr int kPartialFloats = kRowTile * (D + 2);  // a partial result: rows x D, maxima, sums
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T, int D>
__global__ void __launch_bounds__(kRowsThreads, 2) attention_rows_kernel(const AttnParams a) {
    using C = RowsCfg<D>;
    constexpr int kChunks = D / 8;              // 16-byte chunks of a key
    constexpr int kRowsPerPass = 32 / kChunks;  // keys that one pass of the warp's lanes copies
    constexpr int kPasses = kStepKeys / kRowsPerPass;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ PlanShared<kRowsThreads> plan;
    __shared__ float warp_max[4][kRowTile], warp_sum[4][kRowTile];
    __shared__ int last_flag;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    pdl_trigger();
    pdl_wait();
    int x0, x1;
    RunMap map;
    Item it;
    if (!plan_run<kRowTile, kRowsKeyTile, kRowsExtra, kRowsThreads>(a, plan, map, x0, x1, it)) return;

    uint8_t *ring = smem + warp * C::kStages * C::kStepBytes;
    const uint32_t ring_addr = smem_u32(ring);
    const int page_mask = (1 << a.c.page_shift) - 1;
    const T *kb = reinterpret_cast<const T *>(a.c.k), *vb = reinterpret_cast<const T *>(a.c.v);

    for (int x = x0; x < x1;) {
        int kt0, kt1;
        const int upto = run_part<kRowsExtra>(it, x, x1, kt0, kt1);
        if (kt0 == kt1) break;  // the run ends within the item's EXTRA part: its tiles are the next CTA's
        const int r0 = it.rt * kRowTile, rows = min(kRowTile, it.rows - r0);

        // queries: A fragments of the 16 rows
        uint32_t qf[D / 16][4];
        int lo[2], hi[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = r0 + g + 8 * j;
            const bool live = r < it.rows;
            const int tok = live ? a.by_group.div(r) : 0, head = live ? it.h * a.group + r - tok * a.group : 0;
            lo[j] = hi[j] = 0;
            if (live) visible_keys(a, it.seq.keys - it.seq.n + tok, it.seq.keys, lo[j], hi[j]);
            const T *src = reinterpret_cast<const T *>(a.q) + (long long)(it.seq.q0 + tok) * a.q_ts + head * a.q_hs + 2 * t;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                qf[k][j] = live ? *reinterpret_cast<const uint32_t *>(src + 16 * k) : 0u;
                qf[k][2 + j] = live ? *reinterpret_cast<const uint32_t *>(src + 16 * k + 8) : 0u;
            }
        }
        float o[D / 8][4];
#pragma unroll
        for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

        const int steps = kt1 - kt0;
        const int *table = a.c.page_table + (long long)it.s * a.c.max_pages;
        const long long head_off = (long long)it.h * a.c.head_stride + (lane % kChunks) * 8;
        // page of this warp's keys in step j; -1 where none of them is seen
        auto page_of = [&](int j) {
            const int key = (kt0 + j) * kRowsKeyTile + warp * kStepKeys;
            if (j >= steps || key >= it.hi || key + kStepKeys <= it.lo) return -1;
            const int page = table[key >> a.c.page_shift];
            if (page < 0 || page >= a.c.n_pages) {
                report_bad_page(a.c);
                return -1;
            }
            return page;
        };
        auto issue = [&](int j, int page) {
            if (j < steps) {
                const int key = (kt0 + j) * kRowsKeyTile + warp * kStepKeys;
                const uint32_t st = ring_addr + (j % C::kStages) * C::kStepBytes;
                const long long off = page < 0 ? 0 : page * a.c.page_stride + (key & page_mask) * a.c.token_stride + head_off;
#pragma unroll
                for (int i = 0; i < kPasses; ++i) {
                    const int row = i * kRowsPerPass + lane / kChunks;
                    const bool live = page >= 0 && key + row >= it.lo && key + row < it.hi;
                    const long long at = live ? off + row * a.c.token_stride : 0;
                    const uint32_t dst = st + row * (D * 2) + (((lane % kChunks) ^ (row & 7)) << 4);
                    cp_async16(dst, kb + at, live);
                    cp_async16(dst + kStepKeys * D * 2, vb + at, live);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        int next_page = page_of(0);
#pragma unroll
        for (int j = 0; j < C::kStages - 1; ++j) {
            const int page = next_page;
            next_page = page_of(j + 1);
            issue(j, page);
        }
        for (int j = 0; j < steps; ++j) {
            asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 2) : "memory");
            __syncwarp();  // every lane's copies have landed, and stage (j - 1) has been read by all
            {
                const int page = next_page;
                next_page = page_of(j + C::kStages);
                issue(j + C::kStages - 1, page);
            }
            const int key = (kt0 + j) * kRowsKeyTile + warp * kStepKeys;
            if (key >= it.hi || key + kStepKeys <= it.lo) continue;
            const uint32_t ks = ring_addr + (j % C::kStages) * C::kStepBytes, vs = ks + kStepKeys * D * 2;
            float s[2][4] = {};
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int row = n * 8 + (lane & 7);
#pragma unroll
                for (int k = 0; k < D / 32; ++k) {
                    uint32_t b[4];
                    ldmatrix4(ks + row * (D * 2) + (((4 * k + (lane >> 3)) ^ (row & 7)) << 4), b);
                    mma16816<T>(s[n], qf[2 * k], b[0], b[1]);
                    mma16816<T>(s[n], qf[2 * k + 1], b[2], b[3]);
                }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float top = -INFINITY;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int kk = key + n * 8 + 2 * t + e;
                        if (kk < lo[r] || kk >= hi[r]) s[n][2 * r + e] = -INFINITY;
                        top = fmaxf(top, s[n][2 * r + e]);
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float mn = fmaxf(m[r], top);
                const float ref = mn == -INFINITY ? 0.0f : mn * a.scale_log2 - kWeightsUp<T>;
                // of the difference, which is exactly 0 while the maximum stays: a rounded product on one side of a subtraction would
                // multiply the sums by the same number other than one in every step
                const float corr = m[r] == -INFINITY ? 0.0f : exp2f((m[r] - mn) * a.scale_log2);
                m[r] = mn;
                float sum = 0.0f;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float w = exp2f(fmaf(s[n][2 * r + e], a.scale_log2, -ref));
                        s[n][2 * r + e] = w;
                        sum += w;
                    }
                l[r] = l[r] * corr + sum;
#pragma unroll
                for (int n = 0; n < D / 8; ++n) {
                    o[n][2 * r] *= corr;
                    o[n][2 * r + 1] *= corr;
                }
            }
            const uint32_t pf[4] = {Half2Of<T>::pack(s[0][0], s[0][1]), Half2Of<T>::pack(s[0][2], s[0][3]),
                                    Half2Of<T>::pack(s[1][0], s[1][1]), Half2Of<T>::pack(s[1][2], s[1][3])};
            const int vrow = ((lane >> 3) & 1) * 8 + (lane & 7);
#pragma unroll
            for (int n = 0; n < D / 16; ++n) {
                uint32_t b[4];
                ldmatrix4_trans(vs + vrow * (D * 2) + (((2 * n + (lane >> 4)) ^ (vrow & 7)) << 4), b);
                mma16816<T>(o[2 * n], pf, b[0], b[1]);
                mma16816<T>(o[2 * n + 1], pf, b[2], b[3]);
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");

        // join the four warps: each leaves its sums in its part of the ring, then thread = column
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (t == 0) {
                warp_max[warp][g + 8 * r] = m[r];
                warp_sum[warp][g + 8 * r] = l[r];
            }
        }
        __syncthreads();  // all rings drained (rows of one warp's block may lie in another warp's ring)
        float *acc = reinterpret_cast<float *>(smem);
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r)
                *reinterpret_cast<float2 *>(acc + (warp * kRowTile + g + 8 * r) * D + 8 * n + 2 * t) =
                    make_float2(o[n][2 * r], o[n][2 * r + 1]);
        __syncthreads();

        const int begin = it.begin + kRowsExtra;
        const int first = map.run_of(begin), final = map.run_of(begin + (it.kt1 - it.kt0) - 1);
        const bool whole = first == final;
        float *part = a.partials + (long long)(2 * blockIdx.x + ((int)blockIdx.x == first ? 1 : 0)) * C::kPartialFloats;
        for (int i = threadIdx.x; i < rows * (D / 2); i += kRowsThreads) {
            const int r = i / (D / 2), col = 2 * (i % (D / 2));
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < 4; ++w) top = fmaxf(top, warp_max[w][r]);
            float sum = 0.0f;
            float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = warp_max[w][r] == -INFINITY ? 0.0f : exp2f((warp_max[w][r] - top) * a.scale_log2);
                const float2 u = *reinterpret_cast<const float2 *>(acc + (w * kRowTile + r) * D + col);
                sum = fmaf(warp_sum[w][r], f, sum);
                v.x = fmaf(u.x, f, v.x);
                v.y = fmaf(u.y, f, v.y);
            }
            if (whole) {
                const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
                const int rr = r0 + r;
                const int tok = a.by_group.div(rr);
                T *dst = reinterpret_cast<T *>(a.out) + (long long)(it.seq.q0 + tok) * a.o_ts +
                         (long long)(it.h * a.group + rr - tok * a.group) * a.o_hs + col;
                *reinterpret_cast<uint32_t *>(dst) = Half2Of<T>::pack(v.x * inv, v.y * inv);
            } else {
                *reinterpret_cast<float2 *>(part + r * D + col) = v;
                if (col == 0) {
                    part[kRowTile * D + r] = top;
                    part[kRowTile * D + kRowTile + r] = sum;
                }
            }
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                const int before = atomicAdd(a.tickets + first, 1);
                last_flag = before == final - first;
                if (last_flag) a.tickets[first] = 0;  // zero again for the next launch
                __threadfence();
            }
            __syncthreads();
            if (last_flag) {
                // join: all maxima and sums to shared memory, a warp per row turns them into factors, then a thread sums four
                // columns of a row over the parts, several of which are on the way at a time
                __threadfence();
                const int parts = final - first + 1;
                float *factor = reinterpret_cast<float *>(smem), *part_sum = factor + parts * kRowTile;
                auto part_of = [&](int c) {
                    return a.partials + (long long)(2 * (first + c) + (c == 0 ? 1 : 0)) * C::kPartialFloats;
                };
                for (int i = threadIdx.x; i < parts * rows; i += kRowsThreads) {
                    const int c = i / rows, r = i % rows;
                    factor[c * kRowTile + r] = __ldcg(part_of(c) + kRowTile * D + r);
                    part_sum[c * kRowTile + r] = __ldcg(part_of(c) + kRowTile * D + kRowTile + r);
                }
                __syncthreads();
                for (int r = warp; r < rows; r += kRowsThreads / 32) {
                    float top = -INFINITY, sum = 0.0f;
                    for (int c = lane; c < parts; c += 32) top = fmaxf(top, factor[c * kRowTile + r]);
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    const float ref = top == -INFINITY ? 0.0f : top;
                    for (int c = lane; c < parts; c += 32) {
                        const float f = exp2f((factor[c * kRowTile + r] - ref) * a.scale_log2);
                        factor[c * kRowTile + r] = f;
                        sum = fmaf(part_sum[c * kRowTile + r], f, sum);
                    }
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    if (lane == 0) warp_sum[0][r] = sum > 0.0f ? 1.0f / sum : 0.0f;
                }
                __syncthreads();
                for (int i = threadIdx.x; i < rows * (D / 4); i += kRowsThreads) {
                    const int r = i / (D / 4), col = 4 * (i % (D / 4));
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
                    for (int c = 0; c < parts; ++c) {
                        const float4 u = __ldcg(reinterpret_cast<const float4 *>(part_of(c) + r * D + col));
                        const float f = factor[c * kRowTile + r];
                        v.x = fmaf(u.x, f, v.x);
                        v.y = fmaf(u.y, f, v.y);
                        v.z = fmaf(u.z, f, v.z);
                        v.w = fmaf(u.w, f, v.w);
                    }
                    const float inv = warp_sum[0][r];
                    const int rr = r0 + r;
                    const int tok = a.by_group.div(rr);
                    T *dst = reinterpret_cast<T *>(a.out) + (long long)(it.seq.q0 + tok) * a.o_ts +
                             (long long)(it.h * a.group + rr - tok * a.group) * a.o_hs + col;
                    *reinterpret_cast<uint2 *>(dst) =
                        make_uint2(Half2Of<T>::pack(v.x * inv, v.y * inv), Half2Of<T>::pack(v.z * inv, v.w * inv));
                }
            }
        }
        __syncthreads();  // the ring and the warp statistics are free again
        x = upto;
        if (x < x1) next_item<kRowTile, kRowsKeyTile, kRowsExtra>(a, it);
    }
}

struct AttnDeviceInfo {
    int sms = 0;
    bool attr_set[2][2] = {};
};
AttnDeviceInfo &attn_device_info(int dev) {
    static AttnDeviceInfo info[64];
    return info[dev & 63];
}

template <typename T, int D>
int launch_rows(const AttnParams &a, int sms, bool &attr_set, cudaStream_t stream) {
    if (raise_smem_limit(attr_set, attention_rows_kernel<T, D>, RowsCfg<D>::kSmemBytes, "attention_rows")) return 1;
    launch_kernel(attention_rows_kernel<T, D>, dim3(2 * sms), dim3(kRowsThreads), RowsCfg<D>::kSmemBytes, stream, a);
    return check_launch("paged_attention (rows)");
}

int current_device_sms(int &dev) {
    static std::mutex mu;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        dev = 0;
        cudaGetLastError();
    }
    std::lock_guard<std::mutex> lock(mu);
    AttnDeviceInfo &di = attn_device_info(dev);
    if (di.sms == 0 && cudaDeviceGetAttribute(&di.sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        cudaGetLastError();
        di.sms = 0;
        return 148;
    }
    return di.sms;
}

}  // namespace

static size_t workspace_bytes_for(int d_head, int sms) {
    const size_t rows = 4ull * sms * kRowTile * (d_head + 2) * sizeof(float);
    return kTicketBytes + std::max(rows, attention_chunk_partial_bytes(d_head, sms));
}

size_t paged_attention_workspace_size(int d_head) {
    int dev;
    return workspace_bytes_for(d_head, std::min(current_device_sms(dev), kMaxSms));
}

// At most so many units of work; the kernels count them in 32 bits.
static bool work_fits(const b200_w8a8_kv_cache *cache, const b200_w8a8_kv_batch *batch, int group, int row_tile, int key_tile,
                      int extra) {
    const double rows = (double)batch->n_tokens * group / row_tile + batch->n_seqs;
    const double keys = (double)batch->max_pages * cache->page_tokens / key_tile + 1 + extra;
    return rows * keys * cache->n_kv_heads < 2147483000.0;
}

// What a call refuses whatever its rows; 1 after a message.
int check_paged_attention(const b200_w8a8_kv_cache *cache, const b200_w8a8_kv_batch *batch, int n_heads, float scale,
                          int causal_block, int window, const void *workspace, size_t workspace_bytes) {
    if (const char *why = check_paged_cache(cache, batch)) return fail("paged_attention: %s", why);
    if (n_heads <= 0 || n_heads % cache->n_kv_heads != 0)
        return fail("paged_attention: %d heads are no multiple of the cache's %d", n_heads, cache->n_kv_heads);
    if (!(scale > 0.0f) || !isfinite(scale)) return fail("paged_attention: scale must be positive and finite");
    if (causal_block < 0 || window < 0 || (window > 0 && causal_block == 0))
        return fail("paged_attention: causal_block=%d window=%d (a window needs causal_block)", causal_block, window);
    if (batch->n_tokens == 0 || batch->n_seqs == 0) return 0;
    if (((long long)batch->n_tokens * n_heads) >> 30) return fail("paged_attention: n_tokens * n_heads must stay below 2^30");
    const size_t need = paged_attention_workspace_size(cache->d_head);
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < need)
        return fail("paged_attention needs a 256-byte aligned workspace of %zu bytes, got %zu", need,
                    workspace ? workspace_bytes : (size_t)0);
    if (!work_fits(cache, batch, n_heads / cache->n_kv_heads, kChunkRows, kKeyTile, kChunkExtra))
        return fail("paged_attention: %d new tokens over up to %lld keys are too much for one call; pass fewer at a time",
                    batch->n_tokens, (long long)batch->max_pages * cache->page_tokens);
    return 0;
}

int paged_attention(const b200_w8a8_kv_cache *cache, const b200_w8a8_kv_batch *batch, const void *q, long long q_ts,
                    long long q_hs, void *out, long long o_ts, long long o_hs, int n_heads, float scale, int causal_block,
                    int window, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    if (check_paged_attention(cache, batch, n_heads, scale, causal_block, window, workspace, workspace_bytes)) return 1;
    if (batch->n_tokens == 0 || batch->n_seqs == 0) return 0;
    if (!q || !out) return fail("paged_attention: null q or out");
    if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u) || ((q_ts | q_hs | o_ts | o_hs) & 7))
        return fail("paged_attention needs 16-byte aligned q and out and strides that are multiples of 8 elements");
    int dev;
    const int sms = std::min(current_device_sms(dev), kMaxSms);
    AttnParams a{};
    a.c = make_view(cache, batch);
    a.q = q; a.q_ts = q_ts; a.q_hs = q_hs;
    a.out = out; a.o_ts = o_ts; a.o_hs = o_hs;
    a.group = n_heads / cache->n_kv_heads;
    a.by_group.set((unsigned)a.group);
    a.by_block.set((unsigned)std::max(causal_block, 1));
    a.by_heads.set((unsigned)cache->n_kv_heads);
    a.scale_log2 = scale * 1.4426950408889634f;
    a.block = causal_block;
    a.window = window;
    a.tickets = reinterpret_cast<int *>(workspace);
    a.partials = reinterpret_cast<float *>(reinterpret_cast<char *>(workspace) + kTicketBytes);
    AttnDeviceInfo &di = attn_device_info(dev);
    const bool bf = cache->dtype == B200_DT_BF16;
    // One row tile of 16 rows: the rows kernel, bound by HBM whatever the group.  More rows would read every key again for each
    // row tile: measured with 20, 32 and 48 rows, the chunk kernel / the rows kernel, 49.7 / 52.0, 35.1 / 42.5 and 84 / 160 us.
    // What a bound above the real numbers costs: 64 sequences x 1 token, 4 heads a key head, with a bound of 64 / of 1, 334 / 246 us
    // over up to 8191 keys of 128, 77 / 44 us over up to 1000.
    const bool few = (long long)batch->max_new_tokens * a.group <= kRowTile;
    a.min_tiles = 2;  // measured 2 / 4 / 8 / 16 units at least: one sequence of 777 keys 9.7 / 11.2 / 13.8 / 18.9 us
    if (!few || !work_fits(cache, batch, a.group, kRowTile, kRowsKeyTile, kRowsExtra))
        return launch_attention_chunk(cache, a, sms, dev, stream);
    if (cache->d_head == 64)
        return bf ? launch_rows<__nv_bfloat16, 64>(a, sms, di.attr_set[0][1], stream)
                  : launch_rows<__half, 64>(a, sms, di.attr_set[0][0], stream);
    return bf ? launch_rows<__nv_bfloat16, 128>(a, sms, di.attr_set[1][1], stream)
              : launch_rows<__half, 128>(a, sms, di.attr_set[1][0], stream);
}

}  // namespace b200
