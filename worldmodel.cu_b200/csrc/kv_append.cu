// Appends the new keys and values of a batch to the paged cache, with the RMSNorm of each query and key head and the
// position rotation in the same pass:
//     y = x / sqrt(mean(x^2) + eps) * w,     (a, b) -> (a cos - b sin, b cos + a sin)     per rotation pair,
// in fp32, rounded once to the cache's 16-bit type.  Values are only rounded.  Stands in for the ring upsert of the
// reference (src/world_cuda.cu:1898-1960) behind wm_cuda_qkv_fused_rms_rope_i32_dequant (src/world_cuda_ops.cu:1229-1305).
//
// Every element is read once and written once: memory bound.  A head's d elements are spread over d / 8 lanes, 16 bytes of
// output each, so the sum of squares and the exchange of pairs that lie half a head apart are shuffles.  A CTA owns a few
// whole tokens: where they go (sequence, position, page) is found once per token by comparing all sequences' ranges in
// parallel -- two dependent loads instead of a search per head.
#include "paged_kv.cuh"

namespace b200 {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kMaxTokensPerCta = 16;

struct AppendParams {
    KvView c;
    const void *q, *k, *v;
    long long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
    void *q_out;
    long long qo_ts, qo_hs;
    int n_heads;  // of q; 0 without q
    int norm;
    float eps;
    const float *q_weight, *k_weight, *cos, *sin;
    int by_position, rope_rows;
    int tokens_per_cta;
};

struct Place {
    long long kv_offset;  // element offset of (page, 0, slot), < 0: not appended
    int rope_row;         // < 0: the token is left out altogether
};

template <typename TX>
__device__ __forceinline__ void load8(const void *base, long long at, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<float>(const void *base, long long at, float (&x)[8]) {
    const float4 *p = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(base) + at);
    const float4 a = p[0], b = p[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void unpack8(const uint4 &r, float (&x)[8]) {
    float2 f;
    f = Half2Of<T>::unpack(r.x); x[0] = f.x; x[1] = f.y;
    f = Half2Of<T>::unpack(r.y); x[2] = f.x; x[3] = f.y;
    f = Half2Of<T>::unpack(r.z); x[4] = f.x; x[5] = f.y;
    f = Half2Of<T>::unpack(r.w); x[6] = f.x; x[7] = f.y;
}
template <>
__device__ __forceinline__ void load8<__half>(const void *base, long long at, float (&x)[8]) {
    unpack8<__half>(*reinterpret_cast<const uint4 *>(reinterpret_cast<const __half *>(base) + at), x);
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const void *base, long long at, float (&x)[8]) {
    unpack8<__nv_bfloat16>(*reinterpret_cast<const uint4 *>(reinterpret_cast<const __nv_bfloat16 *>(base) + at), x);
}

template <typename TX, typename TC, int D, int ROPE>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const AppendParams p) {
    constexpr int L = D / 8;  // lanes per head
    __shared__ Place place[kMaxTokensPerCta];
    pdl_trigger();
    pdl_wait();
    const int t0 = blockIdx.x * p.tokens_per_cta;
    const int nt = min(p.tokens_per_cta, p.c.n_tokens - t0);
    if ((int)threadIdx.x < nt) place[threadIdx.x] = {-1, -1};
    __syncthreads();
    for (int s = threadIdx.x; s < p.c.n_seqs; s += kAppendThreads) {
        const int q0 = p.c.q_starts[s], q1 = p.c.q_starts[s + 1];
        const int first = max(q0, t0), last = min(q1, t0 + nt);
        for (int t = first; t < last; ++t) {
            const int pos = p.c.kv_lens[s] - (q1 - t);
            if (pos < 0) continue;
            const int index = pos >> p.c.page_shift;
            int page = -1;
            if (index < p.c.max_pages) page = p.c.page_table[(long long)s * p.c.max_pages + index];
            Place at;
            at.rope_row = p.by_position ? pos : t;
            at.kv_offset = -1;
            if (page < 0 || page >= p.c.n_pages || (ROPE != B200_ROPE_NONE && at.rope_row >= p.rope_rows)) {
                report_bad_page(p.c);
                continue;
            }
            at.kv_offset = page * p.c.page_stride + (pos & ((1 << p.c.page_shift) - 1)) * p.c.token_stride;
            place[t - t0] = at;
        }
    }
    __syncthreads();

    const int heads = p.n_heads + 2 * p.c.n_kv_heads;
    const int units = nt * heads;
    const int lane = threadIdx.x % L;
    // every warp runs whole iterations, so the shuffles below have all their lanes
    constexpr int kUnitsPerWarp = 32 / L, kUnitsPerCta = kAppendThreads / L;
    for (int base = (threadIdx.x / 32) * kUnitsPerWarp; base < units; base += kUnitsPerCta) {
        const int unit = base + (threadIdx.x % 32) / L;
        const int tok = min(unit / heads, nt - 1), head = unit % heads;
        const Place at = place[tok];
        const bool live = unit < units && at.kv_offset >= 0;
        const long long t = t0 + tok;
        const bool is_q = head < p.n_heads, is_v = head >= p.n_heads + p.c.n_kv_heads;
        const int h = is_q ? head : is_v ? head - p.n_heads - p.c.n_kv_heads : head - p.n_heads;
        float x[8] = {};
        if (live) {
            if (is_q) load8<TX>(p.q, t * p.q_ts + h * p.q_hs + lane * 8, x);
            else if (is_v) load8<TX>(p.v, t * p.v_ts + h * p.v_hs + lane * 8, x);
            else load8<TX>(p.k, t * p.k_ts + h * p.k_hs + lane * 8, x);
        }
        if (p.norm) {
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (!is_v) {
                const float inv = rsqrtf(ss * (1.0f / D) + p.eps);
                const float *w = is_q ? p.q_weight : p.k_weight;
                if (w) {
                    const float4 a = *reinterpret_cast<const float4 *>(w + lane * 8);
                    const float4 b = *reinterpret_cast<const float4 *>(w + lane * 8 + 4);
                    x[0] *= a.x; x[1] *= a.y; x[2] *= a.z; x[3] *= a.w;
                    x[4] *= b.x; x[5] *= b.y; x[6] *= b.z; x[7] *= b.w;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= inv;
            }
        }
        TC *dst;
        if (is_q) dst = reinterpret_cast<TC *>(p.q_out) + t * p.qo_ts + h * p.qo_hs;
        else dst = reinterpret_cast<TC *>(is_v ? p.c.v : p.c.k) + at.kv_offset + h * p.c.head_stride;
        if (ROPE == B200_ROPE_HALVES) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = __shfl_xor_sync(0xffffffffu, x[j], L / 2);
            if (live && !is_v) {
                const long long row = (long long)at.rope_row * (D / 2) + (lane % (L / 2)) * 8;
                const float sign = lane < L / 2 ? -1.0f : 1.0f;
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const float4 c = *reinterpret_cast<const float4 *>(p.cos + row + 4 * g);
                    const float4 s = *reinterpret_cast<const float4 *>(p.sin + row + 4 * g);
                    x[4 * g + 0] = fmaf(sign * y[4 * g + 0], s.x, x[4 * g + 0] * c.x);
                    x[4 * g + 1] = fmaf(sign * y[4 * g + 1], s.y, x[4 * g + 1] * c.y);
                    x[4 * g + 2] = fmaf(sign * y[4 * g + 2], s.z, x[4 * g + 2] * c.z);
                    x[4 * g + 3] = fmaf(sign * y[4 * g + 3], s.w, x[4 * g + 3] * c.w);
                }
            }
        } else if (ROPE != B200_ROPE_NONE && live && !is_v) {
            const long long row = (long long)at.rope_row * (D / 2) + lane * 4;
            const float4 c = *reinterpret_cast<const float4 *>(p.cos + row);
            const float4 s = *reinterpret_cast<const float4 *>(p.sin + row);
            const float cc[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float a = x[2 * j], b = x[2 * j + 1];
                x[2 * j] = fmaf(-b, sn[j], a * cc[j]);
                x[2 * j + 1] = fmaf(a, sn[j], b * cc[j]);
            }
        }
        if (!live) continue;
        if (ROPE == B200_ROPE_SPLIT && !is_v) {
            *reinterpret_cast<uint2 *>(dst + lane * 4) =
                make_uint2(Half2Of<TC>::pack(x[0], x[2]), Half2Of<TC>::pack(x[4], x[6]));
            *reinterpret_cast<uint2 *>(dst + D / 2 + lane * 4) =
                make_uint2(Half2Of<TC>::pack(x[1], x[3]), Half2Of<TC>::pack(x[5], x[7]));
        } else {
            *reinterpret_cast<uint4 *>(dst + lane * 8) =
                make_uint4(Half2Of<TC>::pack(x[0], x[1]), Half2Of<TC>::pack(x[2], x[3]), Half2Of<TC>::pack(x[4], x[5]),
                           Half2Of<TC>::pack(x[6], x[7]));
        }
    }
}

template <typename TX, typename TC, int D>
cudaError_t launch_append(const AppendParams &p, int rope, dim3 grid, cudaStream_t st) {
    switch (rope) {
        case B200_ROPE_SPLIT: return launch_kernel(kv_append_kernel<TX, TC, D, B200_ROPE_SPLIT>, grid, dim3(kAppendThreads), 0, st, p);
        case B200_ROPE_HALVES: return launch_kernel(kv_append_kernel<TX, TC, D, B200_ROPE_HALVES>, grid, dim3(kAppendThreads), 0, st, p);
        case B200_ROPE_PAIRS: return launch_kernel(kv_append_kernel<TX, TC, D, B200_ROPE_PAIRS>, grid, dim3(kAppendThreads), 0, st, p);
        default: return launch_kernel(kv_append_kernel<TX, TC, D, B200_ROPE_NONE>, grid, dim3(kAppendThreads), 0, st, p);
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
    AppendParams p{};
    p.c = make_view(cache, batch);
    p.q = x->q; p.k = x->k; p.v = x->v;
    p.q_ts = x->q_token_stride; p.q_hs = x->q_head_stride; p.k_ts = x->k_token_stride; p.k_hs = x->k_head_stride;
    p.v_ts = x->v_token_stride; p.v_hs = x->v_head_stride;
    p.q_out = x->q_out; p.qo_ts = x->q_out_token_stride; p.qo_hs = x->q_out_head_stride;
    p.n_heads = x->q ? x->n_heads : 0;
    p.norm = x->norm != 0; p.eps = x->eps; p.q_weight = x->q_weight; p.k_weight = x->k_weight;
    p.cos = x->rope_cos; p.sin = x->rope_sin; p.by_position = x->rope_by_position != 0; p.rope_rows = x->rope_rows;
    p.tokens_per_cta = 1;
    const unsigned grid = (unsigned)((batch->n_tokens + p.tokens_per_cta - 1) / p.tokens_per_cta);
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
