// What the append and the attention kernels share: the cache and the batch as kernels see them, the argument checks, and
// the plan that spreads attention's work over the CTAs.
#pragma once

#include <math.h>

#include "common.cuh"
#include "w8a8_internal.h"

namespace b200 {

struct KvView {
    void *k, *v;
    long long page_stride, head_stride, token_stride;
    int n_pages, page_shift, n_kv_heads;
    const int *page_table, *q_starts, *kv_lens;
    int n_seqs, max_pages, n_tokens;
    int *status;
};

namespace {

__device__ __forceinline__ void report_bad_page(const KvView &c) {
    if (c.status && *(volatile int *)c.status == 0) {
        *(volatile int *)c.status = KS_BAD_PAGE;
        __threadfence_system();
    }
}

// Rows [q0, q0 + n) and key count of sequence s.  Whatever the arrays hold, rows stay within the row buffers and keys
// within the page table.
struct Seq {
    int q0, n, keys;
};
__device__ __forceinline__ Seq load_seq(const KvView &c, int s) {
    Seq q;
    q.q0 = min(max(c.q_starts[s], 0), c.n_tokens);
    q.n = min(max(c.q_starts[s + 1], q.q0), c.n_tokens) - q.q0;
    q.keys = max(c.kv_lens[s], 0);
    const long long most = (long long)c.max_pages << c.page_shift;
    if (q.keys > most) {
        report_bad_page(c);
        q.keys = (int)most;
    }
    return q;
}

// nullptr when the pair is usable, else why not.
const char *check_paged_cache(const b200_w8a8_kv_cache *c, const b200_w8a8_kv_batch *b) {
    if (!c || !b || !c->k_pages || !c->v_pages) return "null cache or batch";
    if (c->dtype != B200_DT_F16 && c->dtype != B200_DT_BF16) return "the cache holds fp16 or bf16";
    if (c->d_head != 64 && c->d_head != 128) return "d_head must be 64 or 128";
    if (c->page_tokens < 16 || c->page_tokens > 256 || (c->page_tokens & (c->page_tokens - 1)))
        return "page_tokens must be 16, 32, 64, 128 or 256";
    if (c->n_pages <= 0 || c->n_kv_heads <= 0) return "the cache needs pages and heads";
    if (((reinterpret_cast<uintptr_t>(c->k_pages) | reinterpret_cast<uintptr_t>(c->v_pages)) & 15u) != 0)
        return "k_pages and v_pages must be 16-byte aligned";
    if ((c->page_stride | c->head_stride | c->token_stride) & 7) return "cache strides must be multiples of 8 elements";
    if (c->page_stride <= 0 || c->head_stride <= 0 || c->token_stride < c->d_head) return "cache strides must be positive";
    if (b->n_seqs < 0 || b->n_tokens < 0 || b->max_pages <= 0) return "negative batch sizes";
    if (b->n_seqs > 0 && (!b->page_table || !b->q_starts || !b->kv_lens)) return "null batch arrays";
    if (((long long)b->max_pages * c->page_tokens) >> 31) return "max_pages * page_tokens must stay below 2^31";
    return nullptr;
}

KvView make_view(const b200_w8a8_kv_cache *c, const b200_w8a8_kv_batch *b) {
    KvView v;
    v.k = c->k_pages;
    v.v = c->v_pages;
    v.page_stride = c->page_stride;
    v.head_stride = c->head_stride;
    v.token_stride = c->token_stride;
    v.n_pages = c->n_pages;
    v.page_shift = __builtin_ctz((unsigned)c->page_tokens);
    v.n_kv_heads = c->n_kv_heads;
    v.page_table = b->page_table;
    v.q_starts = b->q_starts;
    v.kv_lens = b->kv_lens;
    v.n_seqs = b->n_seqs;
    v.max_pages = b->max_pages;
    v.n_tokens = b->n_tokens;
    v.status = status_slot(true);
    return v;
}

template <typename T>
struct Half2Of;
template <>
struct Half2Of<__half> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<uint32_t *>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t w) {
        return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    }
};
template <>
struct Half2Of<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t *>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t w) {
        return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w));
    }
};

// two fp32 values per instruction
__device__ __forceinline__ uint64_t pair2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair2(uint64_t v, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

}  // namespace
}  // namespace b200
