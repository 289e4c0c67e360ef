// Parameters of the attention kernels and the plan that spreads their work.
//
// The query rows of one sequence that read the same key head form one matrix: row r = token * group + head within the group.
// A work item is (sequence, row tile, key head); it has as many KV tiles as its rows can see.  All items' KV tiles, laid end
// to end, are cut into equal runs, one per CTA: a long sequence is split over many CTAs, short ones share a CTA, and every
// CTA finishes at the same time whatever the lengths.  Lengths live on the device, so each CTA derives the plan itself (one
// pass over the sequences, a block scan): no planning launch, no host copy of the lengths, replayable in a graph.
// Beginning and ending an item takes time as well: EXTRA units of work stand before its first tile, so that a run of many
// short items is no longer than one of few long ones.
// Items cut by a run's border leave partial results (unnormalised output, running maximum and sum) in the workspace; the
// last contributor, found by a ticket, joins them in order of their keys, so results do not depend on timing.
#pragma once

#include "paged_kv.cuh"

namespace b200 {

// Division of numbers below 2^31 by a number fixed at launch, as a multiplication.
struct FastDiv {
    unsigned mul, shift, d;
    void set(unsigned divisor) {
        d = divisor;
        shift = 0;
        while (shift < 32 && (1ull << shift) < divisor) ++shift;
        mul = (unsigned)(((1ull << 32) * ((1ull << shift) - divisor)) / divisor + 1);
    }
    __device__ __forceinline__ int div(int n) const { return (int)((__umulhi((unsigned)n, mul) + (unsigned)n) >> shift); }
};

struct AttnParams {
    KvView c;
    const void *q;
    long long q_ts, q_hs;
    void *out;
    long long o_ts, o_hs;
    int group;         // query heads per key head
    FastDiv by_group, by_block, by_heads;  // by_block: of 1 where block is 0; by_heads: of the key heads
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

// a / b for a >= 0, b > 0: the short division whenever both fit 32 bits, which all but absurd sizes do
__device__ __forceinline__ long long div_small(long long a, long long b) {
    if ((((unsigned long long)a | (unsigned long long)b) >> 32) == 0) return (unsigned)a / (unsigned)b;
    return a / b;
}

// Cuts `total` units into `runs` runs of equal length, the first `rest` of them one unit longer.
struct RunMap {
    long long each, rest;
    __device__ __forceinline__ void set(long long total, int runs) {
        each = div_small(total, runs);
        rest = total - each * runs;
    }
    __device__ __forceinline__ long long start(int run) const { return run * each + min((long long)run, rest); }
    // the run that holds unit x
    __device__ __forceinline__ int run_of(long long x) const {
        const long long longer = rest * (each + 1);
        return (int)(x < longer ? div_small(x, each + 1) : rest + div_small(x - longer, each));
    }
};

// First key and one past the last key that the token at position p (< keys) sees; empty where p is negative.
__device__ __forceinline__ void visible_keys(const AttnParams &a, int p, int keys, int &lo, int &hi) {
    lo = 0;
    hi = p < 0 ? 0 : keys;
    if (a.block > 0 && p >= 0) {
        const unsigned end = ((unsigned)a.by_block.div(p) + 1u) * (unsigned)a.block;
        hi = (int)min((unsigned)keys, end);
        if (a.window > 0) lo = min(hi, (int)(end > (unsigned)a.window ? min(end - (unsigned)a.window, (unsigned)keys) : 0u));
    }
}

// KV tiles [kt0, kt1) of KT keys (one at least) that the rows r0 .. r1 - 1 of a sequence see between them, and the first
// and one past the last key of that span.
__device__ __forceinline__ void row_tile_keys(const AttnParams &a, const Seq &s, int r0, int r1, int kt, int &kt0, int &kt1,
                                              int &lo, int &hi) {
    const int base = s.keys - s.n;
    const int p1 = base + a.by_group.div(r1 - 1), p0 = max(base + a.by_group.div(r0), 0);
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
    long long begin;   // where the item begins among all items, in units of tiles
};

template <int NT>
struct PlanShared {
    long long warp_sum[NT / 32];
    long long before;  // work before the sequence found
    Seq seq;
    int s;
};

// Work (for one key head, in tiles) of a sequence over all of its row tiles; every lane of the warp calls with its own.
template <int ROWS, int KT, int EXTRA>
__device__ __forceinline__ long long seq_tiles(const AttnParams &a, const Seq &q) {
    const int rows = q.n * a.group, n_rt = (rows + ROWS - 1) / ROWS;
    long long total = 0;
    int kt0, kt1, lo, hi;
    if (n_rt <= 2) {
        for (int rt = 0; rt < n_rt; ++rt) {
            row_tile_keys(a, q, rt * ROWS, min(rows, (rt + 1) * ROWS), KT, kt0, kt1, lo, hi);
            total += kt1 - kt0 + EXTRA;
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
            sum += kt1 - kt0 + EXTRA;
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

__device__ __forceinline__ Seq lane_seq(const AttnParams &a, int s) {
    if (s < a.c.n_seqs) return load_seq(a.c, s);
    return Seq{0, 0, 0};
}

// The run [x0, x1) of this CTA among all work (false when it has none), and the item that unit x0 belongs to.  All threads of
// the block (NT) call it.
template <int ROWS, int KT, int EXTRA, int NT>
__device__ bool plan_run(const AttnParams &a, PlanShared<NT> &sh, RunMap &map, long long &x0, long long &x1, Item &it) {
    const int heads = a.c.n_kv_heads, lane = threadIdx.x & 31;
    const bool few = a.c.n_seqs <= 32;  // every warp sees all sequences and works for itself: no barrier of the block
    long long per_head = 0, incl = 0, mine = 0;
    Seq q;
    if (few) {
        q = lane_seq(a, lane);
        incl = mine = seq_tiles<ROWS, KT, EXTRA>(a, q);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        per_head = __shfl_sync(0xffffffffu, incl, 31);
    } else {
        for (int base = 0; base < a.c.n_seqs; base += NT) {
            q = lane_seq(a, base + (int)threadIdx.x);
            mine = seq_tiles<ROWS, KT, EXTRA>(a, q);
            long long sum;
            incl = block_scan<NT>(mine, sh, &sum);
            per_head += sum;
        }
    }
    const long long total = per_head * heads;
    if (total == 0) return false;
    const int runs = (int)min((long long)gridDim.x, div_small(total + a.min_tiles - 1, a.min_tiles));
    if ((int)blockIdx.x >= runs) return false;
    map.set(total, runs);
    x0 = map.start(blockIdx.x);
    x1 = map.start(blockIdx.x + 1);
    const long long target = x0 >> 31 ? x0 / heads : (long long)a.by_heads.div((int)x0);
    long long at;  // work for one head before the sequence, then before the row tile
    if (few) {
        const int src = __ffs(__ballot_sync(0xffffffffu, mine > 0 && target < incl)) - 1;
        it.s = src;
        it.seq.q0 = __shfl_sync(0xffffffffu, q.q0, src);
        it.seq.n = __shfl_sync(0xffffffffu, q.n, src);
        it.seq.keys = __shfl_sync(0xffffffffu, q.keys, src);
        at = __shfl_sync(0xffffffffu, incl - mine, src);
    } else {
        long long before = 0;
        for (int base = 0; base < a.c.n_seqs; base += NT) {
            long long sum = per_head;
            if (a.c.n_seqs > NT) {  // else this thread still holds its sequence's values
                q = lane_seq(a, base + (int)threadIdx.x);
                mine = seq_tiles<ROWS, KT, EXTRA>(a, q);
                incl = block_scan<NT>(mine, sh, &sum);
            }
            const long long from = before + incl - mine;
            if (mine > 0 && target >= from && target < from + mine) {
                sh.s = base + (int)threadIdx.x;
                sh.seq = q;
                sh.before = from;
            }
            before += sum;
        }
        __syncthreads();
        it.s = sh.s;
        it.seq = sh.seq;
        at = sh.before;
    }
    it.rows = it.seq.n * a.group;
    const int n_rt = (it.rows + ROWS - 1) / ROWS;
    it.rt = 0;
    // the row tile within the sequence: 32 at a time, every warp for itself
    for (int base = 0; n_rt > 1 && base < n_rt; base += 32) {
        int kt0, kt1, lo, hi, n = 0;
        if (base + lane < n_rt) {
            row_tile_keys(a, it.seq, (base + lane) * ROWS, min(it.rows, (base + lane + 1) * ROWS), KT, kt0, kt1, lo, hi);
            n = kt1 - kt0 + EXTRA;
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
    const int n = it.kt1 - it.kt0 + EXTRA;
    it.h = (int)div_small(x0 - at * heads, n);
    it.begin = at * heads + (long long)it.h * n;
    return true;
}

// The item behind `it` in the order of the plan; called only while there is one.
template <int ROWS, int KT, int EXTRA>
__device__ __forceinline__ void next_item(const AttnParams &a, Item &it) {
    it.begin += it.kt1 - it.kt0 + EXTRA;
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

// What the run [x, x1) holds of an item: tiles [t0, t1) of the item, none where only its EXTRA part lies in the run.
template <int EXTRA>
__device__ __forceinline__ long long run_part(const Item &it, long long x, long long x1, int &t0, int &t1) {
    const long long tiles = it.begin + EXTRA, end = tiles + (it.kt1 - it.kt0), upto = min(x1, end);
    t0 = it.kt0 + (int)max(x - tiles, 0ll);
    t1 = it.kt0 + (int)max(upto - tiles, 0ll);
    return upto;
}

// A walk over the items of one CTA's run.
struct Walk {
    Item it;
    long long x, x1, upto;  // place in the run, its end, the end of this item's part of it
    RunMap map;
    int kt0, kt1;           // KV tiles of the item that the run holds; none at the end of the run
    int first, final;       // the CTAs that share the item
    template <int EXTRA>
    __device__ __forceinline__ void locate() {
        kt0 = kt1 = 0;
        if (x >= x1) return;
        upto = run_part<EXTRA>(it, x, x1, kt0, kt1);
        const long long begin = it.begin + EXTRA;
        first = map.run_of(begin);
        final = map.run_of(begin + (it.kt1 - it.kt0) - 1);
    }
    template <int ROWS, int KT, int EXTRA>
    __device__ __forceinline__ void advance(const AttnParams &a) {
        x = upto;
        if (x < x1) next_item<ROWS, KT, EXTRA>(a, it);
        locate<EXTRA>();
    }
};

}  // namespace

}  // namespace b200
