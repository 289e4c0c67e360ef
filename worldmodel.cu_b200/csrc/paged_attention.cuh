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

#include <mutex>

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
    int min_tiles;     // no CTA gets fewer units than this while others have none
    int *tickets;
    float *partials;
};

// ---- paged_attention_chunk.cu
size_t attention_chunk_partial_bytes(int d_head, int sms);
int launch_attention_chunk(const b200_w8a8_kv_cache *cache, const AttnParams &a, int sms, int dev, cudaStream_t stream);

namespace {

// of the chunk kernel, whose units of work the entry counts too
constexpr int kChunkRows = 256;  // two row tiles
constexpr int kKeyTile = 128;
// EXTRA, measured 1 / 2 / 3 / 5 / 8: the prompt 659 / 532 / 469 / 474 / 487 us (its first CTA has 50 items of one to four tiles), 80 rows
// of 16 sequences 33.5 / 31.6 / 30.6 / 29.3 / 28.9 us, the frame 64.5 / 64.0 / 62.9 / 64.1 / 65.5 us
constexpr int kChunkExtra = 3;
constexpr int kTicketBytes = 32768;                // counters at the start of the workspace
constexpr int kMaxSms = kTicketBytes / 4 / (8 * 3);  // the chunk kernel's joining warps have three each

// Raises a kernel's dynamic shared-memory limit on the current device once; the flag is only touched under the mutex.
template <typename Kernel>
int raise_smem_limit(bool &done, Kernel kernel, int bytes, const char *what) {
    static std::mutex mu;
    std::lock_guard<std::mutex> hold(mu);
    if (done) return 0;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return fail("cudaFuncSetAttribute(%s, smem=%d): %s", what, bytes, cudaGetErrorString(e));
    done = true;
    return 0;
}

// Cuts `total` units into `runs` runs of equal length, the first `rest` of them one unit longer.
struct RunMap {
    unsigned each, rest;
    __device__ __forceinline__ void set(unsigned total, unsigned runs) {
        each = total / runs;
        rest = total - each * runs;
    }
    __device__ __forceinline__ int start(unsigned run) const { return (int)(run * each + min(run, rest)); }
    // the run that holds unit x
    __device__ __forceinline__ int run_of(unsigned x) const {
        const unsigned longer = rest * (each + 1);
        const bool in = x < longer;
        return (int)((in ? 0u : rest) + (in ? x : x - longer) / (in ? each + 1 : each));
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
    int begin;         // where the item begins among all items, in units of tiles
};

template <int NT>
struct PlanShared {
    long long warp_sum[NT / 32];
    Seq seq;
    int s, before;  // the sequence found, and the work before it
};

// Work (for one key head, in tiles) of a sequence over all of its row tiles; every lane of the warp calls with its own
// sequence.  Those of one row tile are done first, a lane each; then the others one by one, a row tile per lane.
template <int ROWS, int KT, int EXTRA>
__device__ __forceinline__ long long seq_work(const AttnParams &a, const Seq &q) {
    const int lane = threadIdx.x & 31, n_rt = (q.n * a.group + ROWS - 1) / ROWS;
    unsigned many = __ballot_sync(0xffffffffu, n_rt > 1);
    long long total = 0;
    bool single = true;
#pragma unroll 1
    do {
        const int src = single ? lane : __ffs(many) - 1;
        Seq w;
        w.q0 = 0;
        w.n = __shfl_sync(0xffffffffu, q.n, src);
        w.keys = __shfl_sync(0xffffffffu, q.keys, src);
        const int rows = w.n * a.group, tiles = (rows + ROWS - 1) / ROWS;
        const int last = single ? (tiles == 1 ? 1 : 0) : tiles;
        long long sum = 0;
#pragma unroll 1
        for (int rt = single ? 0 : lane; rt < last; rt += 32) {
            int kt0, kt1, lo, hi;
            row_tile_keys(a, w, rt * ROWS, min(rows, (rt + 1) * ROWS), KT, kt0, kt1, lo, hi);
            sum += kt1 - kt0 + EXTRA;
        }
        if (single) {
            total = sum;
            single = false;
            continue;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == src) total = sum;
        many &= many - 1;
    } while (many);
    return total;
}

__device__ __forceinline__ long long warp_scan(long long v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
    }
    return v;
}

__device__ __forceinline__ void set_row_tile(const AttnParams &a, Item &it, int rows_per_tile, int kt) {
    const int r0 = it.rt * rows_per_tile;
    row_tile_keys(a, it.seq, r0, min(it.rows, r0 + rows_per_tile), kt, it.kt0, it.kt1, it.lo, it.hi);
}

// The run [x0, x1) of this CTA among all work (false when it has none), and the item that unit x0 belongs to.  All threads of
// the block (NT) call it.  Up to 32 sequences every warp plans for itself; more are spread over the block.
template <int ROWS, int KT, int EXTRA, int NT>
__device__ bool plan_run(const AttnParams &a, PlanShared<NT> &sh, RunMap &map, int &x0, int &x1, Item &it) {
    const int heads = a.c.n_kv_heads, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool few = a.c.n_seqs <= 32;
    const int step = few ? 32 : NT, mine_at = few ? lane : (int)threadIdx.x;
    long long per_head = 0, incl = 0, mine = 0;
    int target = -1;
    Seq q = {0, 0, 0};
    // first the sum over all sequences, then (target >= 0) the sequence that holds this CTA's first unit
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
        long long before = 0;
#pragma unroll 1
        for (int base = 0; base < a.c.n_seqs; base += step) {
            const int s = base + mine_at;
            long long sum;
            if (pass == 0 || a.c.n_seqs > step) {  // else this thread still holds its sequence's values
                q = Seq{0, 0, 0};
                if (s < a.c.n_seqs) q = load_seq(a.c, s);
                mine = seq_work<ROWS, KT, EXTRA>(a, q);
                incl = warp_scan(mine);
                sum = __shfl_sync(0xffffffffu, incl, 31);
                if (!few) {
                    __syncthreads();  // the previous round's readers are done
                    if (lane == 31) sh.warp_sum[warp] = incl;
                    __syncthreads();
                    sum = 0;
#pragma unroll 1
                    for (int w = 0; w < NT / 32; ++w) {
                        if (w < warp) incl += sh.warp_sum[w];
                        sum += sh.warp_sum[w];
                    }
                }
            } else {
                sum = per_head;
            }
            if (pass == 1) {
                const long long from = before + incl - mine;
                const bool here = mine > 0 && target >= from && target < from + mine;
                if (few) {
                    const int src = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
                    it.s = src;
                    it.seq.q0 = __shfl_sync(0xffffffffu, q.q0, src);
                    it.seq.n = __shfl_sync(0xffffffffu, q.n, src);
                    it.seq.keys = __shfl_sync(0xffffffffu, q.keys, src);
                    it.begin = __shfl_sync(0xffffffffu, (int)from, src);
                } else if (here) {
                    sh.s = s;
                    sh.seq = q;
                    sh.before = (int)from;
                }
            }
            before += sum;
        }
        if (pass == 0) {
            per_head = before;
            const long long total = per_head * heads;
            if (total == 0) return false;
            if (total >> 31) {  // only row starts that overlap lead here: the host checks the sizes
                report_bad_page(a.c);
                return false;
            }
            const int runs = min((int)gridDim.x, ((int)total - 1) / a.min_tiles + 1);
            if ((int)blockIdx.x >= runs) return false;
            map.set((unsigned)total, (unsigned)runs);
            x0 = map.start(blockIdx.x);
            x1 = map.start(blockIdx.x + 1);
            target = a.by_heads.div(x0);
        }
    }
    if (!few) {
        __syncthreads();
        it.s = sh.s;
        it.seq = sh.seq;
        it.begin = sh.before;
    }
    it.rows = it.seq.n * a.group;
    const int n_rt = (it.rows + ROWS - 1) / ROWS;
    int at = it.begin;  // work for one head before the row tile
    it.rt = 0;
    // the row tile within the sequence: 32 at a time, every warp for itself
#pragma unroll 1
    for (int base = 0; n_rt > 1 && base < n_rt; base += 32) {
        int kt0, kt1, lo, hi, n = 0;
        if (base + lane < n_rt) {
            row_tile_keys(a, it.seq, (base + lane) * ROWS, min(it.rows, (base + lane + 1) * ROWS), KT, kt0, kt1, lo, hi);
            n = kt1 - kt0 + EXTRA;
        }
        const int scan = (int)warp_scan(n);
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
    it.h = (x0 - at * heads) / n;
    it.begin = at * heads + it.h * n;
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
__device__ __forceinline__ int run_part(const Item &it, int x, int x1, int &t0, int &t1) {
    const int tiles = it.begin + EXTRA, upto = min(x1, tiles + (it.kt1 - it.kt0));
    t0 = it.kt0 + max(x - tiles, 0);
    t1 = it.kt0 + max(upto - tiles, 0);
    return upto;
}

// A walk over the items of one CTA's run.
struct Walk {
    Item it;
    int x, x1, upto;        // place in the run, its end, the end of this item's part of it
    RunMap map;
    int kt0, kt1;           // KV tiles of the item that the run holds; none at the end of the run
    int first, final;       // the CTAs that share the item
    template <int EXTRA>
    __device__ __forceinline__ void locate() {
        kt0 = kt1 = 0;
        if (x >= x1) return;
        upto = run_part<EXTRA>(it, x, x1, kt0, kt1);
        const int begin = it.begin + EXTRA;
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
