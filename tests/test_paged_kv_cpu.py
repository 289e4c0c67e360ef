"""Refusals of the paged cache's entry points, and their plain definitions, without a GPU: every bad argument is turned
away on the host, before anything is launched."""
import ctypes

import pytest
import torch

import paged_kv_reference as pr


def structs(pkg, **kw):
    """A cache, a batch and new tokens of made-up aligned addresses that nothing reads."""
    cache = pkg._Cache(4096, 8192, 64 * 64 * 2, 64 * 64, 64, pkg.DT_F16, 8, 64, 2, 64)
    batch = pkg._Batch(4096, 8192, 12288, 1, 4, 1, 1)
    new = pkg._New(q=4096, k=8192, v=12288, q_token_stride=512, q_head_stride=64, k_token_stride=512, k_head_stride=64,
                   v_token_stride=512, v_head_stride=64, x_dtype=pkg.DT_F16, n_heads=4, q_out=16384, q_out_token_stride=256,
                   q_out_head_stride=64)
    for st in (cache, batch, new):
        for name, value in kw.items():
            if hasattr(st, name):
                setattr(st, name, value)
    return cache, batch, new


CACHE = [("k_pages", None, b"null"), ("k_pages", 4104, b"aligned"), ("dtype", 0, b"fp16 or bf16"), ("d_head", 96, b"d_head"),
         ("page_tokens", 48, b"page_tokens"), ("page_tokens", 8, b"page_tokens"), ("page_tokens", 512, b"page_tokens"),
         ("n_pages", 0, b"pages"), ("n_kv_heads", 0, b"heads"), ("token_stride", 68, b"multiples"), ("token_stride", 32, b"positive"),
         ("page_stride", -64, b"positive"), ("page_table", None, b"null"), ("n_seqs", -1, b"negative"), ("n_tokens", -1, b"negative"),
         ("max_pages", 0, b"negative"), ("max_pages", 2 ** 25, b"2\\^31")]


@pytest.mark.parametrize("field,value,why", CACHE)
def test_bad_caches_and_batches_are_refused(pkg, field, value, why):
    lib = pkg.lib()
    cache, batch, new = structs(pkg, **{field: value})
    if field == "max_pages" and value > 0:
        cache.page_tokens = 64
    r = ctypes.byref
    why = why.replace(b"\\", b"")
    assert lib.b200_w8a8_kv_append(r(cache), r(batch), r(new), None) == 1
    assert b"kv_append" in lib.b200_w8a8_last_error() and why in lib.b200_w8a8_last_error()
    assert lib.b200_w8a8_paged_attention(r(cache), r(batch), 4096, 256, 64, 8192, 256, 64, 4, 0.1, 1, 0, 4096, 1 << 30, None) == 1
    assert b"paged_attention" in lib.b200_w8a8_last_error() and why in lib.b200_w8a8_last_error()


@pytest.mark.parametrize("fields,why", [
    (dict(k=None), b"null k or v"), (dict(q_out=None), b"go together"), (dict(n_heads=0), b"go together"),
    (dict(x_dtype=3), b"fp32, fp16 or bf16"), (dict(rope_order=4), b"rope_order"), (dict(rope_order=1), b"both tables"),
    (dict(rope_order=1, rope_cos=4096, rope_sin=4096, rope_rows=0), b"both tables"),
    (dict(rope_order=2, rope_cos=4096, rope_sin=4096, rope_rows=3, n_tokens=4), b"table rows"),
    (dict(norm=1, eps=-1.0), b"eps"), (dict(norm=1, eps=float("nan")), b"eps"), (dict(q_weight=4096), b"without the norm"),
    (dict(k=8200), b"aligned"), (dict(q_out=16392), b"aligned"), (dict(k_token_stride=516), b"16 bytes"),
    (dict(q_head_stride=4), b"16 bytes"), (dict(q_out_head_stride=4), b"16 bytes"), (dict(x_dtype=0, v_head_stride=62), b"16 bytes")])
def test_bad_new_tokens_are_refused(pkg, fields, why):
    lib = pkg.lib()
    cache, batch, new = structs(pkg, **fields)
    assert lib.b200_w8a8_kv_append(ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(new), None) == 1
    assert why in lib.b200_w8a8_last_error()


@pytest.mark.parametrize("change,why", [
    (dict(q=None), b"null q"), (dict(out=8200), b"aligned"), (dict(q_ts=252), b"multiples"), (dict(n_heads=5), b"no multiple"),
    (dict(n_heads=0), b"no multiple"), (dict(scale=0.0), b"scale"), (dict(scale=float("inf")), b"scale"),
    (dict(scale=float("nan")), b"scale"), (dict(block=-1), b"causal_block"), (dict(window=-1), b"causal_block"),
    (dict(block=0, window=8), b"causal_block"), (dict(ws=None), b"workspace"), (dict(ws=4100), b"workspace"),
    (dict(ws_bytes=4096), b"workspace")])
def test_bad_attention_arguments_are_refused(pkg, change, why):
    lib = pkg.lib()
    cache, batch, _ = structs(pkg)
    a = dict(q=4096, q_ts=256, out=8192, n_heads=4, scale=0.125, block=1, window=0, ws=4096, ws_bytes=1 << 30)
    a.update(change)
    assert lib.b200_w8a8_paged_attention(ctypes.byref(cache), ctypes.byref(batch), a["q"], a["q_ts"], 64, a["out"], 256, 64,
                                         a["n_heads"], a["scale"], a["block"], a["window"], a["ws"], a["ws_bytes"], None) == 1
    assert why in lib.b200_w8a8_last_error()


def test_too_many_query_rows_are_refused(pkg):
    lib = pkg.lib()
    cache, batch, _ = structs(pkg, n_tokens=2 ** 28)
    assert lib.b200_w8a8_paged_attention(ctypes.byref(cache), ctypes.byref(batch), 4096, 256, 64, 8192, 256, 64, 4, 0.125, 1, 0,
                                         4096, 1 << 30, None) == 1
    assert b"2^30" in lib.b200_w8a8_last_error()


def test_empty_calls_launch_nothing(pkg):
    lib = pkg.lib()
    for empty in (dict(n_tokens=0), dict(n_seqs=0)):
        cache, batch, new = structs(pkg, **empty)
        assert lib.b200_w8a8_kv_append(ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(new), None) == 0
        assert lib.b200_w8a8_paged_attention(ctypes.byref(cache), ctypes.byref(batch), None, 256, 64, None, 256, 64, 4, 0.125,
                                             1, 0, None, 0, None) == 0


def test_python_wrappers_refuse_cpu_tensors(pkg):
    pages = torch.zeros(2, 1, 16, 64, dtype=torch.float16)
    with pytest.raises(pkg.W8A8Error, match="CUDA"):
        pkg.PagedKVCache(pages, pages.clone())
    with pytest.raises(pkg.W8A8Error, match="shape"):
        pkg.PagedKVCache(pages, pages[:1])
    with pytest.raises(pkg.W8A8Error, match="strides"):
        pkg.PagedKVCache(pages, torch.zeros(2, 16, 1, 64, dtype=torch.float16).transpose(1, 2)[:, :, :16].transpose(2, 3).contiguous().transpose(2, 3))
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(pkg.W8A8Error, match="int32"):
        pkg.PagedBatch(i32.view(1, 2), i32, i32[:1])
    with pytest.raises(pkg.W8A8Error, match="page_table"):
        pkg.PagedBatch(i32.view(1, 2), i32, i32)


def test_the_bounds_of_the_reference_hold_for_a_plain_rounded_evaluation():
    """The bounds that the GPU tests use, against an evaluation that rounds the weights and the output as the kernels may."""
    for dtype in (torch.float16, torch.bfloat16):
        g = torch.Generator().manual_seed(0)
        n, keys, heads, kv, d = 5, 70, 4, 2, 64
        q, k, v = (torch.randn(r, h, d, generator=g).to(dtype) for r, h in ((n, heads), (keys, kv), (keys, kv)))
        mask = pr.seen(n, keys, 1, 40)
        want, bound = pr.attention(q, k, v, mask, 0.125, dtype)
        kk, vv = k.float().repeat_interleave(2, 1), v.float().repeat_interleave(2, 1)
        s = torch.einsum("nhd,khd->hnk", q.float(), kk) * 0.125
        e = (s.masked_fill(~mask, -float("inf")) - s.masked_fill(~mask, -float("inf")).amax(-1, keepdim=True)).exp()
        o = torch.einsum("hnk,khd->nhd", e.to(dtype).float(), vv) / e.sum(-1).T[..., None]
        assert bool(((o.to(dtype).double() - want).abs() <= bound).all())


def test_arguments_packed_as_bytes_have_the_structures_layout(pkg):
    batch = (11, 12, 13, 4, 5, 6, 7)
    assert pkg._pack_batch(*batch) == bytes(pkg._Batch(*batch))
    new = (21, 22, 23, 1, 2, 3, 4, 5, 6, 1, 32, 24, 7, 8, 1, 1e-5, 25, 26, 2, 27, 28, 1, 99)
    assert pkg._pack_new(*new) == bytes(pkg._New(*new))
