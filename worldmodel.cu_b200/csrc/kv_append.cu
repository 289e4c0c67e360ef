// Appends the new keys and values of a batch to the paged cache, with the RMSNorm of each query and key head and the
// position rotation in the same pass:
//     y = x / sqrt(mean(x^2) + eps) * w,     (a, b) -> (a cos - b sin, b cos + a sin)     per rotation pair,
// in fp32, rounded once to the cache's 16-bit type.  Values are only rounded.  Stands in for the ring upsert of the
// reference (src/world_cuda.cu:1898-1960) behind wm_cuda_qkv_fused_rms_rope_i32_dequant (src/world_cuda_ops.cu:1229-1305).
//
// Every element is read once and written once: memory bound.  A head's d elements are spread over d / 8 lanes, 16 bytes of
// output each, so the sum of squares and the exchange of pairs that lie half a head apart are shuffles.  A warp takes whole
// heads of one token, several at a time in flight, and reads the token's table entries once.  With many tokens a warp has a
// token to itself; with few, two, four or the eight warps of a CTA share one.  Each warp finds its token's place by itself, while
// its first heads are on the way: 32 probes at a time into the sequences' starts, then length and page; no barrier.
//
// Measured: 98348 fp16 rows (32 + 2 x 16 heads of 64) 287 to 295 us = 5.6 TB/s, 86 % of a plain copy (issue slots 68 % busy); a
// frame of 512 fp32 rows 3.8 us, 128 bf16 rows of 128 sequences 4.9 us, one row 2.6 us.  With the places looked up by the CTA
// behind barriers, and addresses and arithmetic element by element, the first took 327 us; without several heads in flight 401.
// Four CTAs per SM leave 64 registers a thread, over which the rotation of halves from 16-bit rows spills 4 to 12 bytes.
#include "paged_kv.cuh"

namespace b200 {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendWarps = kAppendThreads / 32;

struct AppendParams {
    KvView c;
    const void *q, *k, *v;
    long long q_ts, k_ts, v_ts;
    int q_hs, k_hs, v_hs;
    void *q_out;
    long long qo_ts;
    int qo_hs, c_hs;  // c_hs: the cache's head stride
    int n_heads;  // of q; 0 without q
    int norm;
    float eps;
    const float *q_weight, *k_weight, *cos, *sin;
    int by_position, rope_rows;
    int warps_per_token;  // 1, 2, 4 or all of a CTA
};

// The sequence whose new tokens hold row t, -1 if none does: the warp probes 32 starts at a time.
__device__ __forceinline__ int last_start(const KvView &c, int t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = c.n_seqs + 1;  // among q_starts[lo .. hi - 1]
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, i = lo + lane * step;
        const int found = __popc(__ballot_sync(0xffffffffu, i < hi && c.q_starts[min(i, c.n_seqs)] <= t));
        if (found == 0) return -1;
        lo += (found - 1) * step;
        hi = min(hi, lo + step);
    }
    return lo < c.n_seqs && c.q_starts[lo] <= t && t < c.q_starts[lo + 1] ? lo : -1;
}

// Eight elements as they lie in memory, and in fp32.
template <typename TX>
struct Raw8 {
    uint4 v;
    __device__ __forceinline__ void load(const TX *p) {
        v = *reinterpret_cast<const uint4 *>(p);
    }
    __device__ __forceinline__ void unpack(uint64_t (&x)[4]) const {
        float2 f;
        f = Half2Of<TX>::unpack(v.x); x[0] = pair2(f.x, f.y);
        f = Half2Of<TX>::unpack(v.y); x[1] = pair2(f.x, f.y);
        f = Half2Of<TX>::unpack(v.z); x[2] = pair2(f.x, f.y);
        f = Half2Of<TX>::unpack(v.w); x[3] = pair2(f.x, f.y);
    }
};
template <>
struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float *p) {
        a = *reinterpret_cast<const float4 *>(p);
        b = *reinterpret_cast<const float4 *>(p + 4);
    }
    __device__ __forceinline__ void unpack(uint64_t (&x)[4]) const {
        x[0] = pair2(a.x, a.y); x[1] = pair2(a.z, a.w);
        x[2] = pair2(b.x, b.y); x[3] = pair2(b.z, b.w);
    }
};
template <typename TX, typename TC, int D, int ROPE>
__global__ void __launch_bounds__(kAppendThreads, 4) kv_append_kernel(const AppendParams p) {
    constexpr int kInFlight = sizeof(TX) == 4 ? 2 : 4;  // 32 bytes of fp32 a lane, 16 of others: 64 bytes on the way
    constexpr int L = D / 8, kHeads = 32 / L;  // lanes per head, heads per warp and pass
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, per_cta = kAppendWarps / p.warps_per_token;
    const int t0 = blockIdx.x * per_cta;
    // a warp's own part of the rows, the first of it on the way while the token's place is looked up
    const int local = warp / p.warps_per_token;
    const int lane = threadIdx.x % L, sub = (threadIdx.x & 31) / L;
    const int first_v = p.n_heads + p.c.n_kv_heads, heads = first_v + p.c.n_kv_heads;
    const int step = p.warps_per_token * kHeads, start = (warp % p.warps_per_token) * kHeads;
    const long long t = min(t0 + local, p.c.n_tokens - 1);
    Raw8<TX> raw[kInFlight];
    const TX *q_row = reinterpret_cast<const TX *>(p.q) + t * p.q_ts + lane * 8;
    const TX *k_row = reinterpret_cast<const TX *>(p.k) + t * p.k_ts + lane * 8;
    const TX *v_row = reinterpret_cast<const TX *>(p.v) + t * p.v_ts + lane * 8;
    auto fetch = [&](int base) {
#pragma unroll
        for (int u = 0; u < kInFlight; ++u) {
            const int head = min(base + u * step + sub, heads - 1);
            if (head < p.n_heads) raw[u].load(q_row + (long long)head * p.q_hs);
            else if (head < first_v) raw[u].load(k_row + (long long)(head - p.n_heads) * p.k_hs);
            else raw[u].load(v_row + (long long)(head - first_v) * p.v_hs);
        }
    };
    fetch(start);
    if (t0 + local >= p.c.n_tokens) return;  // the whole warp, here and below
    // where the token goes: its sequence is the last one that starts at or before it
    const int seq = last_start(p.c, (int)t);
    if (seq < 0) return;
    const int pos = p.c.kv_lens[seq] - (p.c.q_starts[seq + 1] - (int)t);
    if (pos < 0) return;
    const int index = pos >> p.c.page_shift, rope_row = p.by_position ? pos : (int)t;
    const int page = index < p.c.max_pages ? p.c.page_table[(long long)seq * p.c.max_pages + index] : -1;
    if (page < 0 || page >= p.c.n_pages || (ROPE != B200_ROPE_NONE && rope_row >= p.rope_rows)) {
        report_bad_page(p.c);
        return;
    }
    const long long kv_offset =
        page * p.c.page_stride + (pos & ((1 << p.c.page_shift) - 1)) * p.c.token_stride;
    // Of the pairs that this lane turns: HALVES, two vectors of (x, y) pairs of neighbours; else four pairs (a, b), of which
    // (c, c) and (-s, s) are kept
    uint64_t cs[4], sn[4];
    if (ROPE == B200_ROPE_HALVES) {
        const float sign = lane < L / 2 ? -1.0f : 1.0f;
        const long long row = (long long)rope_row * (D / 2) + (lane % (L / 2)) * 8;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const float4 c = *reinterpret_cast<const float4 *>(p.cos + row + 4 * g);
            const float4 s = *reinterpret_cast<const float4 *>(p.sin + row + 4 * g);
            cs[2 * g] = pair2(c.x, c.y); cs[2 * g + 1] = pair2(c.z, c.w);
            sn[2 * g] = pair2(sign * s.x, sign * s.y); sn[2 * g + 1] = pair2(sign * s.z, sign * s.w);
        }
    } else if (ROPE != B200_ROPE_NONE) {
        const long long row = (long long)rope_row * (D / 2) + lane * 4;
        const float4 c = *reinterpret_cast<const float4 *>(p.cos + row), s = *reinterpret_cast<const float4 *>(p.sin + row);
        cs[0] = pair2(c.x, c.x); cs[1] = pair2(c.y, c.y); cs[2] = pair2(c.z, c.z); cs[3] = pair2(c.w, c.w);
        sn[0] = pair2(-s.x, s.x); sn[1] = pair2(-s.y, s.y); sn[2] = pair2(-s.z, s.z); sn[3] = pair2(-s.w, s.w);
    }
    TC *const q_dst = reinterpret_cast<TC *>(p.q_out) + t * p.qo_ts;
    TC *const k_dst = reinterpret_cast<TC *>(p.c.k) + kv_offset, *const v_dst = reinterpret_cast<TC *>(p.c.v) + kv_offset;
    for (int base = start; base < heads; base += kInFlight * step) {
        if (base != start) fetch(base);
#pragma unroll
        for (int u = 0; u < kInFlight; ++u) {
            if (base + u * step >= heads) break;  // warp-uniform
            const int head = base + u * step + sub;
            const bool live = head < heads, is_q = head < p.n_heads, is_v = head >= first_v;
            uint64_t x[4];
            raw[u].unpack(x);
            if (p.norm) {
                const uint64_t sq = add2(fma2(x[0], x[0], mul2(x[1], x[1])), fma2(x[2], x[2], mul2(x[3], x[3])));
                float ss, more;
                unpair2(sq, ss, more);
                ss += more;
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const float inv = is_v ? 1.0f : rsqrtf(ss * (1.0f / D) + p.eps);
                const uint64_t inv2 = pair2(inv, inv);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = mul2(x[j], inv2);
                const float *w = is_q ? p.q_weight : p.k_weight;
                if (w && !is_v) {
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const float4 ww = *reinterpret_cast<const float4 *>(w + lane * 8 + 4 * g);
                        x[2 * g] = mul2(x[2 * g], pair2(ww.x, ww.y));
                        x[2 * g + 1] = mul2(x[2 * g + 1], pair2(ww.z, ww.w));
                    }
                }
            }
            if (ROPE == B200_ROPE_HALVES) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint64_t y = __shfl_xor_sync(0xffffffffu, (unsigned long long)x[j], L / 2);
                    if (!is_v) x[j] = fma2(y, sn[j], mul2(x[j], cs[j]));
                }
            } else if (ROPE != B200_ROPE_NONE && !is_v) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float a, b;
                    unpair2(x[j], a, b);
                    x[j] = fma2(pair2(b, a), sn[j], mul2(x[j], cs[j]));
                }
            }
            if (!live) continue;
            TC *dst;
            if (is_q) dst = q_dst + (long long)head * p.qo_hs;
            else if (!is_v) dst = k_dst + (long long)(head - p.n_heads) * p.c_hs;
            else dst = v_dst + (long long)(head - first_v) * p.c_hs;
            float a[4], b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) unpair2(x[j], a[j], b[j]);
            if (ROPE == B200_ROPE_SPLIT && !is_v) {
                *reinterpret_cast<uint2 *>(dst + lane * 4) =
                    make_uint2(Half2Of<TC>::pack(a[0], a[1]), Half2Of<TC>::pack(a[2], a[3]));
                *reinterpret_cast<uint2 *>(dst + D / 2 + lane * 4) =
                    make_uint2(Half2Of<TC>::pack(b[0], b[1]), Half2Of<TC>::pack(b[2], b[3]));
            } else {
                *reinterpret_cast<uint4 *>(dst + lane * 8) =
                    make_uint4(Half2Of<TC>::pack(a[0], b[0]), Half2Of<TC>::pack(a[1], b[1]), Half2Of<TC>::pack(a[2], b[2]),
                               Half2Of<TC>::pack(a[3], b[3]));
            }
        }
    }
}

template <typename TX, typename TC, int D>
cudaError_t launch_append(const AppendParams &p, int rope, dim3 grid, cudaStream_t st) {
    switch (rope) {
        case B200_ROPE_SPLIT: return launch_kernel(kv_append_kernel<TX, TC, D, B200_ROPE_SPLIT>, grid, kAppendThreads, 0, st, p);
        case B200_ROPE_HALVES: return launch_kernel(kv_append_kernel<TX, TC, D, B200_ROPE_HALVES>, grid, kAppendThreads, 0, st, p);
        case B200_ROPE_PAIRS: return launch_kernel(kv_append_kernel<TX, TC, D, B200_ROPE_PAIRS>, grid, kAppendThreads, 0, st, p);
        default: return launch_kernel(kv_append_kernel<TX, TC, D, B200_ROPE_NONE>, grid, kAppendThreads, 0, st, p);
    }
}
template <typename TC, int D>
cudaError_t launch_append(const AppendParams &p, int x_dtype, int rope, dim3 grid, cudaStream_t st) {
    if (x_dtype == B200_DT_F32) return launch_append<float, TC, D>(p, rope, grid, st);
    if (x_dtype == B200_DT_F16) return launch_append<__half, TC, D>(p, rope, grid, st);
    return launch_append<__nv_bfloat16, TC, D>(p, rope, grid, st);
}

bool misaligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

}  // namespace

int kv_append(const b200_w8a8_kv_cache *cache, const b200_w8a8_kv_batch *batch, const b200_w8a8_kv_new *x,
              cudaStream_t stream) {
    if (const char *why = check_paged_cache(cache, batch)) return fail("kv_append: %s", why);
    if (!x) return fail("kv_append: null tokens");
    if (batch->n_tokens == 0 || batch->n_seqs == 0) return 0;
    if (!x->k || !x->v) return fail("kv_append: null k or v");
    if ((x->q != nullptr) != (x->q_out != nullptr) || (x->q != nullptr) != (x->n_heads > 0))
        return fail("kv_append: q, q_out and n_heads go together (n_heads=%d)", x->n_heads);
    if (x->x_dtype != B200_DT_F32 && x->x_dtype != B200_DT_F16 && x->x_dtype != B200_DT_BF16)
        return fail("kv_append reads fp32, fp16 or bf16, got type %d", x->x_dtype);
    if (x->rope_order < B200_ROPE_NONE || x->rope_order > B200_ROPE_PAIRS)
        return fail("kv_append: unknown rope_order %d", x->rope_order);
    if (x->rope_order != B200_ROPE_NONE && (!x->rope_cos || !x->rope_sin || x->rope_rows <= 0))
        return fail("kv_append: a rotation needs both tables and their rows");
    if (x->rope_order != B200_ROPE_NONE && !x->rope_by_position && x->rope_rows < batch->n_tokens)
        return fail("kv_append: %d table rows for %d tokens", x->rope_rows, batch->n_tokens);
    if (x->norm && !(x->eps >= 0.0f && isfinite(x->eps))) return fail("kv_append: eps must be finite and not negative");
    if (!x->norm && (x->q_weight || x->k_weight)) return fail("kv_append: norm weights without the norm");
    const void *aligned[] = {x->q, x->k, x->v, x->q_out, x->q_weight, x->k_weight, x->rope_cos, x->rope_sin};
    for (const void *p : aligned)
        if (misaligned(p)) return fail("kv_append needs 16-byte aligned pointers");
    const int64_t unit = x->x_dtype == B200_DT_F32 ? 4 : 8;
    const int64_t in_strides = x->k_token_stride | x->k_head_stride | x->v_token_stride | x->v_head_stride |
                               (x->q ? x->q_token_stride | x->q_head_stride : 0);
    if ((in_strides & (unit - 1)) || (x->q && ((x->q_out_token_stride | x->q_out_head_stride) & 7)))
        return fail("kv_append needs strides that are multiples of 16 bytes");
    const int64_t head_strides[] = {x->k_head_stride, x->v_head_stride, cache->head_stride, x->q ? x->q_head_stride : 0,
                                    x->q ? x->q_out_head_stride : 0};
    for (int64_t h : head_strides)
        if (h < 0 || h >> 31) return fail("kv_append needs head strides from 0 to 2^31 - 1 elements, got %lld", (long long)h);
    AppendParams p{};
    p.c = make_view(cache, batch);
    p.q = x->q; p.k = x->k; p.v = x->v;
    p.q_ts = x->q_token_stride; p.q_hs = (int)x->q_head_stride; p.k_ts = x->k_token_stride; p.k_hs = (int)x->k_head_stride;
    p.v_ts = x->v_token_stride; p.v_hs = (int)x->v_head_stride;
    p.q_out = x->q_out; p.qo_ts = x->q_out_token_stride; p.qo_hs = (int)x->q_out_head_stride; p.c_hs = (int)cache->head_stride;
    p.n_heads = x->q ? x->n_heads : 0;
    p.norm = x->norm != 0; p.eps = x->eps; p.q_weight = x->q_weight; p.k_weight = x->k_weight;
    p.cos = x->rope_cos; p.sin = x->rope_sin; p.by_position = x->rope_by_position != 0; p.rope_rows = x->rope_rows;
    // 148 SMs hold 4736 of these warps.  Few rows are spread over them, many are better off with a place looked up once and all
    // heads of a row behind it.  The number of heads does not enter: of few, most of a row's warps have none.  Measured with
    // 8 / 4 / 2 / 1 warps a row (64 heads of 64, fp16; 48 heads of 128, bf16), us:
    //      400 rows   3.9 /  4.6 /  5.6 /  8.0
    //      800 rows   5.8 /  5.0 /  7.4 /  9.0      8.7 /  8.4 / 12.0 / 15.0
    //     1600 rows   8.8 /  7.4 /  7.9 / 12.6     13.6 / 13.0 / 13.3 / 21.1
    //     3200 rows  16.1 / 11.7 / 11.6 / 13.7     25.6 / 21.3 / 20.9 / 24.2
    //     6400 rows  33.0 / 25.3 / 23.5 / 25.0     53.9 / 44.9 / 38.5 / 42.2
    //    12500 rows  64.8 / 48.0 / 44.6 / 42.8    101.7 / 85.0 / 73.8 / 70.2
    const int n = batch->n_tokens;
    p.warps_per_token = n <= 592 ? kAppendWarps : n <= 2368 ? 4 : n <= 9472 ? 2 : 1;
    const int per_cta = kAppendWarps / p.warps_per_token;
    const unsigned grid = (unsigned)((batch->n_tokens + per_cta - 1) / per_cta);
    if (cache->dtype == B200_DT_F16) {
        if (cache->d_head == 64) launch_append<__half, 64>(p, x->x_dtype, x->rope_order, dim3(grid), stream);
        else launch_append<__half, 128>(p, x->x_dtype, x->rope_order, dim3(grid), stream);
    } else {
        if (cache->d_head == 64) launch_append<__nv_bfloat16, 64>(p, x->x_dtype, x->rope_order, dim3(grid), stream);
        else launch_append<__nv_bfloat16, 128>(p, x->x_dtype, x->rope_order, dim3(grid), stream);
    }
    return check_launch("kv_append");
}

}  // namespace b200
