"""Attention over the paged cache at the ends of its numbers: long runs of one CTA, weights far below the largest, values that
are no numbers, scales and head groups away from the usual ones, and how long a wait lasts."""
import pytest
import torch

import paged_kv_reference as pr

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def shared_pages(k, v, page, seqs):
    """A cache that holds the one key / value sequence k, v [keys, kv_heads, d], and a page table by which `seqs` sequences
    all read it."""
    keys, heads, d = k.shape
    pages = -(-keys // page)
    pools = []
    for x in (k, v):
        pool = torch.zeros(pages * page, heads, d, dtype=x.dtype, device=DEV)
        pool[:keys] = x
        pools.append(pool.view(pages, page, heads, d).transpose(1, 2))
    table = torch.arange(pages, dtype=torch.int32, device=DEV).expand(seqs, pages).contiguous()
    return (*pools, table)


# ------------------------------------------------------------------ long runs
@pytest.mark.parametrize("hint", [1, 1000])
def test_a_long_run_of_one_cta_weighs_old_and_new_keys_alike(pkg, hint):
    """592 sequences of 131072 keys over 148 SMs: every CTA walks whole sequences, 2048 steps of 64 keys or 1024 of 128 each.  The
    first 64 keys have the largest score, all others one and the same, log2 of it between 92 and 185 before
    the maximum is taken; products and sums of the scores are exact in fp32.  Values are one in the first half and minus one in
    the second (even columns), or one throughout (odd columns).

    Bound: weights and output are rounded once each, 2^-11 relative (a = sum w |v| = 1); the sums of products and of weights
    take one addition per matrix instruction of 16 keys and accumulator, each off by at most 2^-23 of a sum of one sign, so
    2 x 2^-23 x additions: 2048 (one of four warps, 16 keys each) and 4096 (one of two accumulators); 2^-18 for exponentials and
    joins."""
    seqs, keys, d, page, dtype = 592, 131072, 64, 256, torch.float16
    k = torch.full((keys, 1, d), 4.0, dtype=dtype, device=DEV)
    k[:64, :, 0] = 4.5
    v = torch.ones(keys, 1, d, dtype=dtype, device=DEV)
    v[keys // 2:, :, ::2] = -1.0
    k_pages, v_pages, table = shared_pages(k, v, page, seqs)
    g = torch.Generator().manual_seed(11)
    gain = torch.randint(128, 256, (seqs,), generator=g).to(DEV) / 64.0  # [2, 4), exact in 8 bits
    q = gain[:, None, None].expand(seqs, 1, d).to(dtype).contiguous()
    cache = pkg.PagedKVCache(k_pages, v_pages)
    batch = pkg.PagedBatch(table, torch.arange(seqs + 1, dtype=torch.int32, device=DEV),
                           torch.full((seqs,), keys, dtype=torch.int32, device=DEV), max_new_tokens=hint)
    got = pkg.paged_attention(q, cache, batch).double()[:, 0]
    late = torch.exp(-gain.double() * 0.5 * d ** -0.5)  # weight of a key behind the first 64
    total = 64 + (keys - 64) * late
    even = (64 + (keys // 2 - 64) * late - keys // 2 * late) / total
    additions = 2048 if hint == 1 else 4096
    bound = 2.0 ** -11 * (1 + even.abs()) + 2 * 2.0 ** -23 * additions + 2.0 ** -18
    assert pkg.poll_status() == 0
    off = (got[:, ::2] - even[:, None]).abs().amax(1), (got[:, 1::2] - 1).abs().amax(1)
    print("largest errors", float(off[0].max()), float(off[1].max()))
    assert bool((off[0] <= bound).all()), float(off[0].max())
    assert bool((off[1] <= bound + 2.0 ** -11).all()), float(off[1].max())
