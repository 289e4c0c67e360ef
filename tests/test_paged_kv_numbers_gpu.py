"""Attention over the paged cache at the ends of its numbers: long runs of one CTA, weights far below the largest, values that
are no numbers, scales and head groups away from the usual ones, and how long a wait lasts."""
import math

import pytest
import torch

import paged_kv_reference as pr

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
POLY = {"f16": 2.8e-6, "bf16": 1.0e-4}  # relative error of the exponentials that the chunk kernel computes as polynomials


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


# ------------------------------------------------------------------ weights far below the largest
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hint", [1, 1000])
def test_many_small_weights_beside_a_large_one(pkg, dtype, hint):
    """131071 keys, one of which has a score 18 above all others: the others' weights are 1.5e-8 of the largest, and make 0.002
    of the sum.  Their values are one, the large one's zero in even columns.  592 sequences, so that a CTA has whole ones.

    Bound: half a step for each of the two roundings of normal numbers.  fp16 weights are kept 2^7 times as large at least,
    so that one below the normal range loses 2^-25 / 2^7 of the largest: 131071 x 2^-32.  Sums: at most 8192 additions to
    one accumulator, 2^-23 each, above and below the fraction.  Polynomial exponentials: 1.0e-4 (bf16), 2.8e-6 (fp16), likewise."""
    seqs, keys, d, page, t = 592, 131071, 64, 128, pr.DTYPES[dtype]
    k = torch.zeros(keys, 1, d, dtype=t, device=DEV)
    k[777] = 2.25  # 64 x 2.25 / 8 = 18
    v = torch.ones(keys, 1, d, dtype=t, device=DEV)
    v[777, :, ::2] = 0.0
    k_pages, v_pages, table = shared_pages(k, v, page, seqs)
    q = torch.ones(seqs, 1, d, dtype=t, device=DEV)
    batch = pkg.PagedBatch(table, torch.arange(seqs + 1, dtype=torch.int32, device=DEV),
                           torch.full((seqs,), keys, dtype=torch.int32, device=DEV), max_new_tokens=hint)
    got = pkg.paged_attention(q, pkg.PagedKVCache(k_pages, v_pages), batch).double()
    small = (keys - 1) * math.exp(-18.0)
    want = small / (1 + small)
    lost = keys * 2.0 ** -32 if dtype == "f16" else 0.0
    rel = 2 * pr.half_step(t) + 8192 * 2 * 2.0 ** -23 + 2 * POLY[dtype]
    off = float((got[..., ::2] - want).abs().max()), float((got[..., 1::2] - 1).abs().max())
    print("largest errors", off, "of", want)
    assert pkg.poll_status() == 0
    assert off[0] <= rel * want + lost, off
    assert off[1] <= rel + lost, off


# ------------------------------------------------------------------ no numbers
def formula(q, k, v, mask, scale):
    """softmax in 64 bits as torch has it, over the keys that a token sees; a token none of whose scores is above minus
    infinity gets zeros.  q [n, heads, d], k, v [keys, kv_heads, d]."""
    group = q.shape[1] // k.shape[1]
    q, k, v = (x.double() for x in (q, k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)))
    s = (torch.einsum("nhd,khd->nhk", q, k) * scale).masked_fill(~mask.to(q.device)[:, None], -math.inf)
    nothing = (s == -math.inf).all(-1, keepdim=True)
    w = torch.where(nothing, torch.zeros_like(s), torch.softmax(s, -1))
    return torch.einsum("nhk,khd->nhd", w, v)


@pytest.mark.parametrize("dtype,d", [("f16", 64), ("bf16", 128), ("f16", 128), ("bf16", 64)])
@pytest.mark.parametrize("new,hint", [(1, 1), (40, 1000), (200, 1000)])
@pytest.mark.parametrize("what", ["nan key", "inf key", "nan query", "inf query", "nan value", "inf value"])
def test_what_is_no_number_where_it_is_seen(pkg, dtype, d, new, hint, what):
    """70 sequences, each with one element of one key, value or query that is NaN or infinite, at each place modulo 35 and more.
    Outputs are NaN, infinite or finite where those of the definition are, and finite ones within the usual bound.  An infinite key
    gives scores of plus infinity (no number is left) or minus infinity (a weight of zero) by the query's sign."""
    t, seqs, heads, kv = pr.DTYPES[dtype], 70, 4, 2
    keys = 70 + new
    g = torch.Generator().manual_seed(d + new)
    shapes = [(new, keys)] * seqs
    k_pages, v_pages, table, contents = pr.make_cache(shapes, 32, kv, d, t, "heads", g, DEV, fill=0.0)
    q = torch.randn(seqs, new, heads, d, generator=g).to(t)
    q[q == 0] = 1.0
    bad = math.nan if "nan" in what else math.inf
    for s in range(seqs):
        (k, v), place = contents[s], s
        if "query" in what:
            q[s, s % new, s % heads, s % d] = bad
            continue
        x, pool = (k, k_pages) if "key" in what else (v, v_pages)
        x[place, s % kv, s % d] = bad
        pool[int(table[s, place // 32]), s % kv, place % 32, s % d] = bad
    cache = pkg.PagedKVCache(k_pages, v_pages)
    batch = pkg.PagedBatch(table, pr.starts_of(shapes, DEV), pr.lens_of(shapes, DEV), max_new_tokens=hint)
    got = pkg.paged_attention(q.view(-1, heads, d).to(DEV), cache, batch).view(seqs, new, heads, d)
    assert pkg.poll_status() == 0
    mask = pr.seen(new, keys, 1, 0)
    for s in range(seqs):
        k, v = contents[s]
        want = formula(q[s], k, v, mask, d ** -0.5)
        mine = got[s].cpu()
        assert torch.equal(mine.isnan(), want.isnan()), (s, "NaN")
        assert torch.equal(mine.isinf(), want.isinf()), (s, "infinite")
        assert torch.equal(mine[mine.isinf()].double(), want[want.isinf()]), (s, "sign")
        clean = [x.nan_to_num(0.0, 0.0, 0.0) for x in (q[s], k, v)]
        _, bound = pr.attention(*clean, mask, d ** -0.5, t)
        ok = want.isfinite()
        assert bool(((mine.double() - want).abs() <= 2 * bound)[ok].all()), s


def test_no_score_above_minus_infinity_gives_zeros(pkg):
    d, kv, t = 64, 1, torch.float16
    k = torch.zeros(50, kv, d, dtype=t, device=DEV)
    k[:, :, 0] = -math.inf
    v = torch.ones(50, kv, d, dtype=t, device=DEV)
    k_pages, v_pages, table = shared_pages(k, v, 16, 1)
    for new, hint in ((1, 1), (30, 1000)):
        batch = pkg.PagedBatch(table, torch.tensor([0, new], dtype=torch.int32, device=DEV),
                               torch.tensor([50], dtype=torch.int32, device=DEV), max_new_tokens=hint)
        q = torch.ones(new, 2, d, dtype=t, device=DEV)
        assert bool((pkg.paged_attention(q, pkg.PagedKVCache(k_pages, v_pages), batch) == 0).all())


# ------------------------------------------------------------------ scales and head groups
def definition(q, k, v, n, keys, scale, dtype):
    """The output in 64 bits and its bound, the polynomials' term among it: an error of that size in every weight, in
    numerator and denominator."""
    t, mask = pr.DTYPES[dtype], pr.seen(n, keys, 1, 0)
    want, bound = pr.attention(q, k.to(DEV), v.to(DEV), mask, scale, t)
    return want, bound + 2 * POLY[dtype] * pr.attention(q, k.to(DEV), v.abs().to(DEV), mask, scale, t)[0]


@pytest.mark.parametrize("scale", [1.0, 0.3, 1e-4, 3.0])
@pytest.mark.parametrize("dtype,d", [("f16", 64), ("bf16", 128)])
def test_scales(pkg, scale, dtype, d):
    t, heads, kv, shapes = pr.DTYPES[dtype], 6, 2, [(1, 300), (90, 400), (1, 1), (9, 2000)]
    g = torch.Generator().manual_seed(d)
    k_pages, v_pages, table, contents = pr.make_cache(shapes, 32, kv, d, t, "heads", g, DEV)
    cache, starts = pkg.PagedKVCache(k_pages, v_pages), pr.starts_of(shapes, DEV)
    q = torch.randn(101, heads, d, generator=g).to(t).to(DEV)
    for hint in (1, 1000):
        out = pkg.paged_attention(q, cache, pkg.PagedBatch(table, starts, pr.lens_of(shapes, DEV), max_new_tokens=hint), scale=scale)
        at = 0
        for (n, keys), (k, v) in zip(shapes, contents):
            want, bound = definition(q[at:at + n], k, v, n, keys, scale, dtype)
            assert bool(((out[at:at + n].double() - want).abs() <= bound).all()), (hint, n, keys)
            at += n
    assert pkg.poll_status() == 0


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (9, 3), (5, 1), (14, 2), (16, 1), (40, 2), (48, 1)])
@pytest.mark.parametrize("new", [1, 3, 37])
@pytest.mark.parametrize("dtype,d,order", [("bf16", 128, "tokens"), ("f16", 128, "heads"), ("bf16", 64, "heads")])
def test_head_groups_of_every_kernel(pkg, heads, kv_heads, new, dtype, d, order):
    t, shapes = pr.DTYPES[dtype], [(new, 200), (new, new), (new, 77)]
    g = torch.Generator().manual_seed(heads)
    k_pages, v_pages, table, contents = pr.make_cache(shapes, 64, kv_heads, d, t, order, g, DEV)
    q = torch.randn(3 * new, heads, d, generator=g).to(t).to(DEV)
    batch = pkg.PagedBatch(table, pr.starts_of(shapes, DEV), pr.lens_of(shapes, DEV), max_new_tokens=new)
    out = pkg.paged_attention(q, pkg.PagedKVCache(k_pages, v_pages), batch)
    assert pkg.poll_status() == 0
    for i, ((n, keys), (k, v)) in enumerate(zip(shapes, contents)):
        want, bound = definition(q[i * new:(i + 1) * new], k, v, n, keys, d ** -0.5, dtype)
        assert bool(((out[i * new:(i + 1) * new].double() - want).abs() <= bound).all()), (n, keys)


# ------------------------------------------------------------------ workspaces
@pytest.mark.parametrize("new,keys", [(1, 40000), (32, 60000), (300, 9000)])
def test_of_a_workspace_only_the_counters_have_to_be_zero(pkg, new, keys):
    heads, kv, d = 4, 1, 64
    g = torch.Generator().manual_seed(new)
    k_pages, v_pages, table, _ = pr.make_cache([(new, keys)], 64, kv, d, torch.float16, "heads", g, DEV, fill=0.0)
    cache = pkg.PagedKVCache(k_pages, v_pages)
    batch = pkg.PagedBatch(table, pr.starts_of([(new, keys)], DEV), pr.lens_of([(new, keys)], DEV), max_new_tokens=new)
    q = torch.randn(new, heads, d, generator=g).half().to(DEV)
    clean = pkg.make_attention_workspace(cache)
    clean.zero_()
    dirty = torch.full_like(clean, 255)  # NaN as floats
    dirty[:32768] = 0
    want = pkg.paged_attention(q, cache, batch, workspace=clean)
    assert torch.equal(pkg.paged_attention(q, cache, batch, workspace=dirty), want) and bool(want.isfinite().all())
    assert torch.equal(pkg.paged_attention(q, cache, batch), want)
    assert pkg.poll_status() == 0


# ------------------------------------------------------------------ waits
@pytest.mark.parametrize("limit_ms", [20, 200])
def test_a_wait_lasts_as_long_as_its_limit(pkg, limit_ms):
    """One page load left out by the test switch: the kernel gives up no sooner than the limit says, and soon after it."""
    L = pkg.lib()
    seqs, heads, kv, d = [(300, 2000), (40, 64)], 4, 2, 64
    g = torch.Generator().manual_seed(1)
    k_pages, v_pages, table, _ = pr.make_cache(seqs, 32, kv, d, torch.float16, "heads", g, DEV)
    cache = pkg.PagedKVCache(k_pages, v_pages)
    batch = pkg.PagedBatch(table, pr.starts_of(seqs, DEV), pr.lens_of(seqs, DEV))
    q = torch.randn(340, heads, d, generator=g).half().to(DEV)
    ws = pkg.make_attention_workspace(cache)
    want = pkg.paged_attention(q, cache, batch, workspace=ws)
    torch.cuda.synchronize()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    try:
        L.b200_w8a8_debug_set_wait_limit_ns(limit_ms * 1_000_000)
        L.b200_w8a8_debug_drop_operand_load(1)
        begin.record()
        pkg.paged_attention(q, cache, batch, workspace=ws)
        end.record()
        torch.cuda.synchronize()
        took = begin.elapsed_time(end)
        with pytest.raises(pkg.W8A8Error, match="gave up a bounded wait"):
            pkg.paged_attention(q, cache, batch, workspace=ws)
    finally:
        L.b200_w8a8_debug_drop_operand_load(0)
        L.b200_w8a8_debug_set_wait_limit_ns(0)
    print("limit", limit_ms, "ms, took", took)
    ws.zero_()
    assert torch.equal(pkg.paged_attention(q, cache, batch, workspace=ws), want)
    assert pkg.poll_status() == 0
    assert limit_ms <= took <= 4 * limit_ms + 100


# ------------------------------------------------------------------ types
@pytest.mark.parametrize("dtype", [torch.float64, torch.int64, torch.uint8, torch.float8_e4m3fn, torch.float32, torch.int32])
def test_other_types_are_refused(pkg, dtype):
    pages = torch.zeros(2, 1, 16, 64, device=DEV)
    x = torch.zeros(1, 1, 64, device=DEV)
    batch = pkg.PagedBatch(*(torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([[0]], [0, 1], [1])))
    with pytest.raises(pkg.W8A8Error):
        pkg.kv_append(pkg.PagedKVCache(pages.to(dtype), pages.to(dtype)), batch, x, x)
    if dtype != torch.float32:
        with pytest.raises(pkg.W8A8Error):
            pkg.kv_append(pkg.PagedKVCache(pages.half(), pages.half()), batch, x.to(dtype), x.to(dtype))
