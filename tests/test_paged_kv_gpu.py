"""The paged key / value cache on the GPU: append (norm, rotation, places) and attention against their definitions in 64
bits, with bounds derived from the roundings; pages outside a sequence hold NaN, unused table entries hold no pages."""
import pytest
import torch

import paged_kv_reference as pr

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def run_attention(pkg, seqs, heads, kv_heads, d, page, dtype, order="heads", block=1, window=0, seed=0, hint=None,
                  tail_rows=3, gain=1.5, cache_edit=None):
    dtype = pr.DTYPES[dtype]
    g = torch.Generator().manual_seed(seed)
    k_pages, v_pages, table, contents = pr.make_cache(seqs, page, kv_heads, d, dtype, order, g, DEV)
    if cache_edit:
        cache_edit(k_pages, v_pages, table)
    rows = sum(n for n, _ in seqs)
    q = (torch.randn(rows + tail_rows, heads, d, generator=g) * gain).to(dtype)
    out = torch.full(q.shape, 7.0, dtype=dtype, device=DEV)
    cache = pkg.PagedKVCache(k_pages, v_pages)
    batch = pkg.PagedBatch(table, pr.starts_of(seqs, DEV), pr.lens_of(seqs, DEV), max_new_tokens=hint)
    ws = pkg.make_attention_workspace(cache)
    pkg.paged_attention(q.to(DEV), cache, batch, causal_block=block, window=window, out=out, workspace=ws)
    again = torch.full_like(out, 7.0)
    pkg.paged_attention(q.to(DEV), cache, batch, causal_block=block, window=window, out=again, workspace=ws)
    torch.cuda.synchronize()
    assert pkg.poll_status() == 0
    assert int(ws[:32768].count_nonzero()) == 0, "the workspace's counters are zero after a call"
    assert torch.equal(out, again), "the same call twice gives the same bits"
    at = 0
    for (n, keys), (k, v) in zip(seqs, contents):
        want, bound = pr.attention(q[at:at + n].to(DEV), k.to(DEV), v.to(DEV), pr.seen(n, keys, block, window), d ** -0.5,
                                   dtype)
        got = out[at:at + n].double()
        assert torch.isfinite(got).all(), (n, keys)
        over = (got - want).abs() - bound
        assert float(over.max() if over.numel() else 0.0) <= 0, (n, keys, float((got - want).abs().max()), float(over.max()))
        at += n
    assert bool((out[at:] == 7.0).all()), "rows behind the last sequence are left as they were"
    return out


EDGES = [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300]


@pytest.mark.parametrize("dtype,d,order", [("f16", 64, "heads"), ("bf16", 128, "tokens"), ("f16", 128, "heads"),
                                           ("bf16", 64, "tokens")])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_single_tokens_at_every_edge(pkg, dtype, d, order, page):
    seqs = [(min(1, n), n) for n in EDGES]
    run_attention(pkg, seqs, 8, 4, d, page, dtype, order, seed=page)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (2, 1), (9, 3), (5, 1), (7, 1), (14, 2), (16, 1), (40, 2), (48, 1), (3, 3)])
@pytest.mark.parametrize("new", [1, 3, 37])
def test_head_groups(pkg, heads, kv_heads, new):
    run_attention(pkg, [(new, 200), (new, new), (new, 77)], heads, kv_heads, 64, 16, "f16", seed=heads)


@pytest.mark.parametrize("dtype,d,page,order", [("f16", 64, 64, "heads"), ("bf16", 128, 16, "tokens"),
                                                ("f16", 128, 128, "tokens"), ("bf16", 64, 32, "heads"),
                                                ("bf16", 128, 256, "heads")])
@pytest.mark.parametrize("block,window", [(1, 0), (0, 0), (1, 100), (64, 0), (50, 120), (33, 5), (1, 1), (10 ** 9, 0)])
def test_chunks_of_ragged_sequences(pkg, dtype, d, page, order, block, window):
    seqs = [(130, 130), (0, 50), (1, 1), (257, 700), (64, 64), (5, 513), (0, 0), (128, 300), (200, 1025)]
    run_attention(pkg, seqs, 8, 4, d, page, dtype, order, block, window, seed=block % 1000 + window)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("block", [0, 1, 40])
def test_fewer_keys_than_new_tokens(pkg, d, block):
    """Tokens at negative positions see nothing and get zeros."""
    out = run_attention(pkg, [(5, 2), (300, 100), (3, 0), (1, 0), (2, 2)], 4, 2, d, 16, "f16", block=block)
    assert bool((out[:3] == 0).all()) and bool((out[5:205] == 0).all()) and bool((out[305:309] == 0).all())


@pytest.mark.parametrize("hint", [None, 1, 10 ** 6])
def test_the_bound_on_new_tokens_only_chooses_the_kernel(pkg, hint):
    run_attention(pkg, [(1, 40), (300, 900), (17, 64)], 8, 2, 128, 32, "bf16", hint=hint)


@pytest.mark.parametrize("new,keys,heads,kv_heads", [(1, 20011, 8, 1), (1, 5000, 32, 8), (4, 9001, 16, 2), (600, 3001, 4, 2),
                                                     (512, 8704, 4, 2), (20, 30001, 4, 2), (3, 20000, 8, 1)])
def test_one_sequence_over_the_whole_machine(pkg, new, keys, heads, kv_heads):
    """The key axis is split and the parts joined."""
    run_attention(pkg, [(new, keys)], heads, kv_heads, 64, 64, "f16", block=512 if new == 512 else 1)
    run_attention(pkg, [(new, keys)], heads, kv_heads, 128, 16, "bf16", "tokens")


@pytest.mark.parametrize("seqs", [400, 1100])
def test_many_sequences(pkg, seqs):
    run_attention(pkg, [(i % 3, i % 3 + 7 * i % 90) for i in range(seqs)], 4, 2, 64, 16, "bf16")


def test_pages_that_a_window_has_left_may_be_gone(pkg):
    seqs, page, window = [(1, 900), (40, 1000), (1, 333)], 16, 130

    def edit(k_pages, v_pages, table):
        for s, (n, keys) in enumerate(seqs):
            first = max(0, keys - n + 1 - window)  # of the first new token
            table[s, :first // page] = -1
    run_attention(pkg, seqs, 4, 2, 128, page, "f16", window=window, cache_edit=edit)


def test_peaked_and_even_scores(pkg):
    run_attention(pkg, [(3, 1000), (200, 700)], 4, 2, 128, 32, "f16", gain=30.0)
    run_attention(pkg, [(3, 1000), (200, 700)], 4, 2, 128, 32, "bf16", gain=1e-3)


def test_strided_queries_and_outputs(pkg):
    """q as a slice of fused QKV rows, out head-major."""
    seqs, heads, kv, d = [(70, 170), (1, 33)], 4, 2, 64
    g = torch.Generator().manual_seed(1)
    k_pages, v_pages, table, contents = pr.make_cache(seqs, 32, kv, d, torch.float16, "tokens", g, DEV)
    rows = torch.randn(71, (heads + 2 * kv) * d, generator=g).half().to(DEV)
    q = rows.view(71, -1, d)[:, :heads]
    out = torch.zeros(heads, 71, d, dtype=torch.float16, device=DEV)
    cache = pkg.PagedKVCache(k_pages, v_pages)
    batch = pkg.PagedBatch(table, pr.starts_of(seqs, DEV), pr.lens_of(seqs, DEV))
    pkg.paged_attention(q, cache, batch, out=out.transpose(0, 1))
    dense = pkg.paged_attention(q.contiguous(), cache, batch)
    torch.cuda.synchronize()
    assert torch.equal(out.transpose(0, 1), dense)


def test_offsets_beyond_32_bits(pkg):
    """A pool of more than 2^31 elements, its last pages in use."""
    page, kv, d = 256, 16, 128
    pages = 2 ** 31 // (page * kv * d) + 40
    k_pages, v_pages = (torch.full((pages, kv, page, d), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    seqs = [(1, 700), (150, 600)]
    g = torch.Generator().manual_seed(5)
    table = torch.tensor([[pages - 1, pages - 2, pages - 3], [pages - 7, 3, pages - 5]], dtype=torch.int32, device=DEV)
    q = torch.randn(151, 32, d, generator=g).bfloat16().to(DEV)
    k, v = (torch.randn(151, kv, d, generator=g).bfloat16().to(DEV) for _ in range(2))
    for s, (n, keys) in enumerate(seqs):
        for i in range(3):
            for pool in (k_pages, v_pages):
                pool[int(table[s, i])] = torch.randn(kv, page, d, generator=g).bfloat16().to(DEV)
    cache = pkg.PagedKVCache(k_pages, v_pages)
    batch = pkg.PagedBatch(table, pr.starts_of(seqs, DEV), pr.lens_of(seqs, DEV))
    pkg.kv_append(cache, batch, k, v)
    out = pkg.paged_attention(q, cache, batch)
    at = 0
    for s, (n, keys) in enumerate(seqs):
        own = [pool[table[s].long()].transpose(1, 2).reshape(-1, kv, d)[:keys] for pool in (k_pages, v_pages)]
        assert torch.equal(own[0][keys - n:], k[at:at + n]) and torch.equal(own[1][keys - n:], v[at:at + n])
        want, bound = pr.attention(q[at:at + n], *own, pr.seen(n, keys, 1, 0), d ** -0.5, torch.bfloat16)
        assert bool(((out[at:at + n].double() - want).abs() <= bound).all())
        at += n
    assert pkg.poll_status() == 0


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("x,dtype", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f16")])
@pytest.mark.parametrize("d,page,order,rope,by_position,norm,weights",
                         [(64, 16, "heads", "split", False, True, False), (128, 64, "tokens", "halves", True, True, True),
                          (64, 128, "tokens", "halves", False, False, False), (128, 32, "heads", "pairs", True, True, False),
                          (64, 256, "heads", "pairs", False, True, True), (128, 16, "heads", "split", True, False, False),
                          (64, 64, "tokens", "none", False, True, True), (128, 128, "heads", "none", False, False, False)])
def test_append(pkg, x, dtype, d, page, order, rope, by_position, norm, weights):
    seqs, heads, kv = [(3, 3), (0, 20), (1, 1), (17, 40), (1, 129), (0, 0), (40, 300), (5, 2), (33, 65)], 6, 2
    dtype, xt = pr.DTYPES[dtype], pr.DTYPES[x]
    g = torch.Generator().manual_seed(d + page)
    k_pages, v_pages, table, contents = pr.make_cache(seqs, page, kv, d, dtype, order, g, DEV, fill=5.0)
    rows, spare = sum(n for n, _ in seqs), 4
    src = (torch.randn(rows + spare, heads + 2 * kv, d, generator=g) * 3).to(xt).to(DEV)
    q, k, v = src[:, :heads], src[:, heads:heads + kv], src[:, heads + kv:]
    table_rows = 400 if by_position else rows + spare
    angle = torch.rand(table_rows, d // 2, generator=g) * 6.3
    cos, sin = angle.cos().to(DEV), angle.sin().to(DEV)
    qw, kw = ((1 + 0.2 * torch.randn(d, generator=g)).to(DEV) if weights else None for _ in range(2))
    order_code = {"none": None, "split": pkg.ROPE_SPLIT, "halves": pkg.ROPE_HALVES, "pairs": pkg.ROPE_PAIRS}[rope]
    want = [p.clone() for p in (k_pages, v_pages)]
    q_out = torch.full((rows + spare, heads, d), 9.0, dtype=dtype, device=DEV)
    cache = pkg.PagedKVCache(k_pages, v_pages)
    batch = pkg.PagedBatch(table, pr.starts_of(seqs, DEV), pr.lens_of(seqs, DEV))
    args = dict(norm_eps=1e-5 if norm else None, q_weight=qw, k_weight=kw, rope_cos=cos if order_code else None,
                rope_sin=sin if order_code else None, rope_order=order_code, rope_by_position=by_position)
    assert pkg.kv_append(cache, batch, k, v, q=q, q_out=q_out, **args) is q_out
    torch.cuda.synchronize()
    assert pkg.poll_status() == 0
    # fp32 work: the sum of squares of d terms, a reciprocal square root, three products and a sum; 16 half steps of fp32
    # cover them relative to the absolute terms of an element; then one rounding to the cache's type
    fp32 = 16 * 2.0 ** -24
    at = 0
    for s, (n, keys) in enumerate(seqs):
        for i in range(n):
            t, pos = at + i, keys - n + i
            if pos < 0:
                assert bool((q_out[t] == 9.0).all())
                continue
            row = pos if by_position else t
            where = (int(table[s, pos // page]), slice(None), pos % page)
            for part, w, got in ((q, qw, q_out[t]), (k, kw, k_pages[where])):
                y, terms = pr.append(part[t:t + 1], args["norm_eps"], w, rope, cos[row:row + 1], sin[row:row + 1])
                tol = pr.half_step(dtype) * y.abs() * (1 + 2.0 ** -10) + fp32 * terms + pr.tiny_step(dtype)
                assert bool(((got.double() - y[0]).abs() <= tol[0]).all()), (s, i)
            assert torch.equal(v_pages[where], v[t].to(dtype))
            want[0][where], want[1][where] = k_pages[where], v_pages[where]
        at += n
    assert torch.equal(k_pages, want[0]) and torch.equal(v_pages, want[1]), "nothing else of the cache changed"
    assert bool((q_out[rows:] == 9.0).all())
    # without queries the cache gets the same
    k2, v2 = (torch.full_like(p, 5.0) for p in (k_pages, v_pages))
    del args["q_weight"]
    assert pkg.kv_append(pkg.PagedKVCache(k2, v2), batch, k, v, **args) is None
    torch.cuda.synchronize()
    at = 0
    for s, (n, keys) in enumerate(seqs):
        for pos in range(max(0, keys - n), keys):
            where = (int(table[s, pos // page]), slice(None), pos % page)
            assert torch.equal(k2[where], k_pages[where]) and torch.equal(v2[where], v_pages[where])


@pytest.mark.parametrize("seqs,new", [(1, 2000), (300, 1), (7, 101), (1000, 3), (5, 2603)])
def test_append_many(pkg, seqs, new):
    """Every token at its place, many sequences or many tokens (values only: bit for bit)."""
    d, kv, page = 64, 3, 16
    lens = [(new, new + 5 * i % 23) for i in range(seqs)]
    g = torch.Generator().manual_seed(seqs)
    k_pages, v_pages, table, contents = pr.make_cache(lens, page, kv, d, torch.float16, "heads", g, DEV, fill=0.0)
    rows = seqs * new
    k, v = (torch.randn(rows, kv, d, generator=g).half().to(DEV) for _ in range(2))
    want = [p.clone() for p in (k_pages, v_pages)]
    s = torch.arange(rows, device=DEV) // new
    pos = torch.tensor([n for _, n in lens], device=DEV)[s] - new + torch.arange(rows, device=DEV) % new
    for pool, x in zip(want, (k, v)):
        pool[table.long()[s, pos // page], :, pos % page] = x
    pkg.kv_append(pkg.PagedKVCache(k_pages, v_pages), pkg.PagedBatch(table, pr.starts_of(lens, DEV), pr.lens_of(lens, DEV)),
                  k, v)
    torch.cuda.synchronize()
    assert torch.equal(k_pages, want[0]) and torch.equal(v_pages, want[1])


@pytest.mark.parametrize("x,d,rope", [("f32", 64, "SPLIT"), ("bf16", 128, "HALVES"), ("f16", 128, "PAIRS")])
def test_append_in_parts(pkg, x, d, rope):
    """However many rows a call has, and however its warps share them, a row comes out the same bit for bit."""
    heads, kv, page, rows = 5, 3, 32, 13001
    g = torch.Generator().manual_seed(d)
    dtype = torch.float16 if x == "f16" else torch.bfloat16
    k_pages, v_pages, table, _ = pr.make_cache([(rows, rows + 9)], page, kv, d, dtype, "tokens", g, DEV, fill=0.0)
    src = torch.randn(rows, heads + 2 * kv, d, generator=g).to(pr.DTYPES[x]).to(DEV)
    angle = torch.rand(rows + 9, d // 2, generator=g) * 6.3
    kw = dict(norm_eps=1e-5, rope_order=getattr(pkg, "ROPE_" + rope), rope_cos=angle.cos().to(DEV), rope_sin=angle.sin().to(DEV),
              rope_by_position=True)
    got = {}
    for part in (500, 2000, 9001, rows):
        pools = [torch.zeros_like(k_pages), torch.zeros_like(v_pages)]
        q_out = torch.zeros(rows, heads, d, dtype=dtype, device=DEV)
        cache = pkg.PagedKVCache(*pools)
        for a in range(0, rows, part):
            b = min(rows, a + part)
            batch = pkg.PagedBatch(table, torch.tensor([0, b - a], dtype=torch.int32, device=DEV),
                                   torch.tensor([b + 9], dtype=torch.int32, device=DEV))
            pkg.kv_append(cache, batch, src[a:b, heads:heads + kv], src[a:b, heads + kv:], q=src[a:b, :heads], q_out=q_out[a:b], **kw)
        torch.cuda.synchronize()
        assert pkg.poll_status() == 0
        got[part] = (q_out, *pools)
    for part in got:
        assert all(torch.equal(a, b) for a, b in zip(got[part], got[rows])), part


# ------------------------------------------------------------------ streams, graphs, errors
def test_a_captured_step_follows_the_lengths_on_the_device(pkg):
    """Append and attention of one token captured once, replayed while the lengths grow."""
    heads, kv, d, page = 4, 2, 64, 16
    g = torch.Generator().manual_seed(3)
    k_pages, v_pages = (torch.randn(12, kv, page, d, generator=g).half().to(DEV) for _ in range(2))
    table = torch.arange(12, dtype=torch.int32).view(2, 6).to(DEV)
    lens = torch.tensor([30, 60], dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    rows = torch.randn(2, heads + 2 * kv, d, generator=g).half().to(DEV)
    cache, batch = pkg.PagedKVCache(k_pages, v_pages), pkg.PagedBatch(table, starts, lens, max_new_tokens=1)
    ws = pkg.make_attention_workspace(cache)
    q_out, out = torch.empty(2, heads, d, dtype=torch.float16, device=DEV), torch.empty(2, heads, d, dtype=torch.float16, device=DEV)

    def step():
        pkg.kv_append(cache, batch, rows[:, heads:heads + kv], rows[:, heads + kv:], q=rows[:, :heads], q_out=q_out, norm_eps=1e-6)
        pkg.paged_attention(q_out, cache, batch, out=out, workspace=ws)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for _ in range(5):
        lens += 1
        rows.copy_(torch.randn(rows.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for s in range(2):
            n = int(lens[s])
            own = [p[table[s].long()].transpose(1, 2).reshape(-1, kv, d)[:n] for p in (k_pages, v_pages)]
            assert torch.equal(own[1][-1], rows[s, heads + kv:])
            want, bound = pr.attention(q_out[s:s + 1], *own, pr.seen(1, n, 1, 0), d ** -0.5, torch.float16)
            assert bool(((out[s:s + 1].double() - want).abs() <= bound).all())
    assert pkg.poll_status() == 0


def test_two_streams_with_a_workspace_each(pkg):
    heads, kv, d = 8, 2, 128
    streams, jobs = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(2):
        seqs = [(1, 6000 + i), (90, 500)]
        g = torch.Generator().manual_seed(i)
        k_pages, v_pages, table, _ = pr.make_cache(seqs, 32, kv, d, torch.bfloat16, "heads", g, DEV)
        cache = pkg.PagedKVCache(k_pages, v_pages)
        batch = pkg.PagedBatch(table, pr.starts_of(seqs, DEV), pr.lens_of(seqs, DEV))
        q = torch.randn(91, heads, d, generator=g).bfloat16().to(DEV)
        jobs.append((q, cache, batch, pkg.make_attention_workspace(cache), pkg.paged_attention(q, cache, batch)))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, (q, cache, batch, ws, _) in enumerate(jobs):
            with torch.cuda.stream(streams[i]):
                outs[i].append(pkg.paged_attention(q, cache, batch, workspace=ws))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, jobs[i][4]) for o in outs[i])


def test_pages_and_lengths_outside_the_cache_are_reported_once(pkg):
    """A bad page in use, a length beyond the table: nothing is accessed there, the next call returns an error once."""
    heads, kv, d, page = 4, 2, 64, 16
    pages = torch.zeros(4, kv, page, d, dtype=torch.float16, device=DEV)
    starts = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    x = torch.ones(1, heads + 2 * kv, d, dtype=torch.float16, device=DEV)

    def call(table, length, what, new=1):
        cache = pkg.PagedKVCache(pages, pages.clone())
        b = pkg.PagedBatch(torch.tensor([table], dtype=torch.int32, device=DEV), starts,
                           torch.tensor([length], dtype=torch.int32, device=DEV), max_new_tokens=new)
        if what == "append":
            return pkg.kv_append(cache, b, x[:, heads:heads + kv], x[:, heads + kv:])
        return pkg.paged_attention(x[:, :heads].contiguous(), cache, b)
    for what in ("append", "attend"):
        for table, length in (([4, 0], 3), ([-1, 0], 16), ([0, 1], 33), ([0, 2 ** 30], 17), ([0, 1], 2 ** 31 - 1)):
            for new in (1, 1000):
                call(table, length, what, new)
                torch.cuda.synchronize()
                with pytest.raises(pkg.W8A8Error, match="outside its cache"):
                    call([0, 1], 3, what)
                call([0, 1], 3, what)
                torch.cuda.synchronize()
                assert pkg.poll_status() == 0


def test_a_wait_that_runs_out_is_reported_once(pkg):
    """One page load left out by the test switch: the kernel gives up after 5 ms, drains and returns; the next call says so
    once; with the workspace zeroed again everything is as before."""
    L = pkg.lib()
    seqs, heads, kv, d = [(300, 2000), (40, 64)], 4, 2, 128
    g = torch.Generator().manual_seed(1)
    k_pages, v_pages, table, _ = pr.make_cache(seqs, 32, kv, d, torch.float16, "heads", g, DEV)
    cache = pkg.PagedKVCache(k_pages, v_pages)
    batch = pkg.PagedBatch(table, pr.starts_of(seqs, DEV), pr.lens_of(seqs, DEV))
    q = torch.randn(340, heads, d, generator=g).half().to(DEV)
    ws = pkg.make_attention_workspace(cache)
    want = pkg.paged_attention(q, cache, batch, workspace=ws)
    torch.cuda.synchronize()
    try:
        L.b200_w8a8_debug_set_wait_limit_ns(5_000_000)
        L.b200_w8a8_debug_drop_operand_load(1)
        pkg.paged_attention(q, cache, batch, workspace=ws)
        torch.cuda.synchronize()
        with pytest.raises(pkg.W8A8Error, match="gave up a bounded wait"):
            pkg.paged_attention(q, cache, batch, workspace=ws)
    finally:
        L.b200_w8a8_debug_drop_operand_load(0)
        L.b200_w8a8_debug_set_wait_limit_ns(0)
    ws.zero_()
    assert torch.equal(pkg.paged_attention(q, cache, batch, workspace=ws), want)
    torch.cuda.synchronize()
    assert pkg.poll_status() == 0
