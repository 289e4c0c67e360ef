// Parameters of the attention kernels and the plan that spreads their work.
//
// The query rows of one sequence that read the same key head form one matrix: row r = token * group + head within the group.
// A work item is (sequence, row tile, key head); it has as many KV tiles as its rows can see.  All items' KV tiles, laid end
// to end, are cut into equal runs, one per CTA: a long sequence is split over many CTAs, short ones share a CTA, and every
// CTA finishes at the same time whatever the lengths.  Lengths live on the device, so each CTA derives the plan itself (one
// pass over the sequences, a block scan): no planning launch, no host copy of the lengths, replayable in a graph.
// Items cut by a run's border leave partial results (unnormalised output, running maximum and sum) in the workspace; the
// last contributor, found by a ticket, joins them in order of their keys, so results do not depend on timing.
#pragma once

#include "paged_kv.cuh"

namespace b200 {

struct AttnParams {
    KvView c;
    const void *q;
    long long q_ts, q_hs;
    void *out;
    long long o_ts, o_hs;
    int group;         // query heads per key head
    float scale_log2;  // scale * log2(e): weights are 2^(scale_log2 * (s - max))
    int block, window;
    int min_tiles;     // no CTA gets fewer KV tiles than this while others have none
    int *tickets;
    float *partials;
};

// ---- paged_attention_chunk.cu
size_t attention_chunk_partial_bytes(int d_head, int sms);
int launch_attention_chunk(const b200_w8a8_kv_cache *cache, const AttnParams &a, int sms, int dev, cudaStream_t stream);

namespace {

constexpr int kTicketBytes = 16384;           // counters at the start of the workspace: one per warp that joins
constexpr int kMaxSms = kTicketBytes / 4 / 8;  // eight such warps per SM

// First key and one past the last key that the token at position p (< keys) sees; empty where p is negative.
__device__ __forceinline__ void visible_keys(const AttnParams &a, int p, int keys, int &lo, int &hi) {
    lo = 0;
    hi = p < 0 ? 0 : keys;
    if (a.block > 0 && p >= 0) {
        const unsigned end = ((unsigned)p / (unsigned)a.block + 1u) * (unsigned)a.block;
        hi = (int)min((unsigned)keys, end);
        if (a.window > 0) lo = min(hi, (int)(end > (unsigned)a.window ? min(end - (unsigned)a.window, (unsigned)keys) : 0u));
    }
}

// KV tiles [kt0, kt1) of KT keys (one at least) that the rows r0 .. r1 - 1 of a sequence see between them, and the first
// and one past the last key of that span.
__device__ __forceinline__ void row_tile_keys(const AttnParams &a, const Seq &s, int r0, int r1, int kt, int &kt0, int &kt1,
                                              int &lo, int &hi) {
    const int base = s.keys - s.n;
    const int p1 = base + (r1 - 1) / a.group, p0 = max(base + r0 / a.group, 0);
    int l, h;
    visible_keys(a, p1, s.keys, l, h);
    hi = h;
    if (p1 >= 0) {
        visible_keys(a, p0, s.keys, l, h);
        lo = min(l, hi);
    } else {
        lo = 0;
    }
    kt0 = lo / kt;
    kt1 = max(kt0 + 1, (hi + kt - 1) / kt);
}

struct Item {
    int s, rt, h;      // sequence, row tile, key head
    Seq seq;
    int rows;          // of the sequence: new tokens * group
    int kt0, kt1;      // KV tiles
    int lo, hi;        // keys
    long long begin;   // index of the item's first tile among all tiles
};

template <int NT>
struct PlanShared {
    long long warp_sum[NT / 32];
    long long before;  // tiles before the sequence found
    int s, rt;
};

// Tiles (for one key head) of sequence s over all of its row tiles; every lane of the warp calls with its own sequence.
template <int ROWS, int KT>
__device__ __forceinline__ long long seq_tiles(const AttnParams &a, int s) {
    Seq q = {0, 0, 0};
    if (s < a.c.n_seqs) q = load_seq(a.c, s);
    const int rows = q.n * a.group, n_rt = (rows + ROWS - 1) / ROWS;
    long long total = 0;
    int kt0, kt1, lo, hi;
    if (n_rt <= 2) {
        for (int rt = 0; rt < n_rt; ++rt) {
            row_tile_keys(a, q, rt * ROWS, min(rows, (rt + 1) * ROWS), KT, kt0, kt1, lo, hi);
            total += kt1 - kt0;
        }
    }
    // sequences of many row tiles: the warp takes them together, a row tile per lane
    unsigned many = __ballot_sync(0xffffffffu, n_rt > 2);
    const int lane = threadIdx.x & 31;
    while (many) {
        const int src = __ffs(many) - 1;
        many &= many - 1;
        Seq w;
        w.q0 = 0;
        w.n = __shfl_sync(0xffffffffu, q.n, src);
        w.keys = __shfl_sync(0xffffffffu, q.keys, src);
        const int wrows = w.n * a.group, wn = (wrows + ROWS - 1) / ROWS;
        long long sum = 0;
        for (int rt = lane; rt < wn; rt += 32) {
            row_tile_keys(a, w, rt * ROWS, min(wrows, (rt + 1) * ROWS), KT, kt0, kt1, lo, hi);
            sum += kt1 - kt0;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == src) total = sum;
    }
    return total;
}

// Inclusive scan of `v` over the block; *sum gets the block's total.
template <int NT>
__device__ __forceinline__ long long block_scan(long long v, PlanShared<NT> &sh, long long *sum) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
    }
    __syncthreads();  // the previous round's readers are done
    if (lane == 31) sh.warp_sum[warp] = v;
    __syncthreads();
    long long all = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
        if (w < warp) v += sh.warp_sum[w];
        all += sh.warp_sum[w];
    }
    *sum = all;
    return v;
}

__device__ __forceinline__ void set_row_tile(const AttnParams &a, Item &it, int rows_per_tile, int kt) {
    const int r0 = it.rt * rows_per_tile;
    row_tile_keys(a, it.seq, r0, min(it.rows, r0 + rows_per_tile), kt, it.kt0, it.kt1, it.lo, it.hi);
}

// The run [x0, x1) of this CTA among all tiles (false when it has none), and the item that tile x0 belongs to.  `runs` gets
// the number of CTAs that have work, `total` the number of tiles.  All threads of the block (NT) call it.
template <int ROWS, int KT, int NT>
__device__ bool plan_run(const AttnParams &a, PlanShared<NT> &sh, long long &total, int &runs, long long &x0, long long &x1,
                         Item &it) {
    const int heads = a.c.n_kv_heads;
    long long per_head = 0, incl = 0, mine = 0;
    for (int base = 0; base < a.c.n_seqs; base += NT) {
        mine = seq_tiles<ROWS, KT>(a, base + (int)threadIdx.x);
        long long sum;
        incl = block_scan<NT>(mine, sh, &sum);
        per_head += sum;
    }
    total = per_head * heads;
    if (total == 0) return false;
    const long long wanted = (total + a.min_tiles - 1) / a.min_tiles;
    runs = (int)min((long long)gridDim.x, wanted);
    if ((int)blockIdx.x >= runs) return false;
    x0 = blockIdx.x * total / runs;
    x1 = (blockIdx.x + 1) * total / runs;
    const long long target = x0 / heads;
    long long before = 0;
    for (int base = 0; base < a.c.n_seqs; base += NT) {
        long long sum = per_head;
        if (a.c.n_seqs > NT) {  // else this thread still holds its sequence's values
            mine = seq_tiles<ROWS, KT>(a, base + (int)threadIdx.x);
            incl = block_scan<NT>(mine, sh, &sum);
        }
        const long long from = before + incl - mine;
        if (mine > 0 && target >= from && target < from + mine) {
            sh.s = base + (int)threadIdx.x;
            sh.before = from;
        }
        before += sum;
    }
    __syncthreads();
    it.s = sh.s;
    it.seq = load_seq(a.c, it.s);
    it.rows = it.seq.n * a.group;
    long long at = sh.before;
    const int n_rt = (it.rows + ROWS - 1) / ROWS, lane = threadIdx.x & 31;
    it.rt = 0;
    // the row tile within the sequence: 32 at a time, every warp for itself
    for (int base = 0; base < n_rt; base += 32) {
        int kt0, kt1, lo, hi, n = 0;
        if (base + lane < n_rt) {
            row_tile_keys(a, it.seq, (base + lane) * ROWS, min(it.rows, (base + lane + 1) * ROWS), KT, kt0, kt1, lo, hi);
            n = kt1 - kt0;
        }
        long long scan = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += up;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, n > 0 && target < at + scan);
        if (hit) {
            const int src = __ffs(hit) - 1;
            it.rt = base + src;
            at += __shfl_sync(0xffffffffu, scan - n, src);
            break;
        }
        at += __shfl_sync(0xffffffffu, scan, 31);
    }
    set_row_tile(a, it, ROWS, KT);
    const int n = it.kt1 - it.kt0;
    it.h = (int)((x0 - at * heads) / n);
    it.begin = at * heads + (long long)it.h * n;
    return true;
}

// The item behind `it` in the order of the plan; called only while there is one.
template <int ROWS, int KT>
__device__ __forceinline__ void next_item(const AttnParams &a, Item &it) {
    it.begin += it.kt1 - it.kt0;
    if (++it.h < a.c.n_kv_heads) return;
    it.h = 0;
    if (++it.rt * ROWS >= it.rows) {
        it.rt = 0;
        do {
            if (++it.s >= a.c.n_seqs) return;
            it.seq = load_seq(a.c, it.s);
        } while (it.seq.n == 0);
        it.rows = it.seq.n * a.group;
    }
    set_row_tile(a, it, ROWS, KT);
}

// The CTA whose run holds tile x.
__device__ __forceinline__ int run_of(long long x, long long total, int runs) {
    return (int)(((x + 1) * runs - 1) / total);
}

}  // namespace

}  // namespace b200
