"""A whole layer over the paged cache in one call (b200_w8a8_layer_forward_paged): it equals the composition of the public
operators bit for bit, frame after frame; and it agrees with the two-call form around an attention in 64 bits."""
import pytest
import torch

import paged_kv_reference as pr
from test_layer_driver_gpu import frame, make_layer, slab

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1.1920929e-07


def setup(pkg, T, D, HQ, HKV, DH, HID, ctrl, use_slab, page, dtype, worlds, seed=3):
    host = make_layer(D, HQ, HKV, DH, HID, seed, ctrl)
    layout = pkg.W_SLAB128 if use_slab else pkg.W_ROW_MAJOR
    L = {k: (slab(v) if (use_slab and k.startswith("w_")) else v).to(DEV) for k, v in host.items()}
    pages = worlds * (-(-4 * T // page))
    k_pages, v_pages = (torch.full((pages, HKV, page, DH), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(pages, generator=g).view(worlds, -1).to(torch.int32).to(DEV)
    drv = pkg.ReferenceLayerDriver(worlds * T, D, HQ, HKV, DH, HID, EPS, w_layout=layout)
    return L, layout, pkg.PagedKVCache(k_pages, v_pages), table, drv, g


def composition(pkg, L, layout, tokens, cos, sin, cache, batch, HQ, HKV, DH, block, window, ws):
    lin = lambda q, s, w, sw, **kw: pkg.linear(q, s, L[w], L[sw], n=L[sw].shape[0], w_layout=layout, out_dtype=torch.float32, **kw)
    q1, s1 = pkg.rms_norm_quantize_rows(tokens, L["mod_scale0"], L["mod_bias0"], EPS, scale_is_mod=True)
    x = lin(q1, s1, "w_qkv", "s_qkv").view(tokens.shape[0], HQ + 2 * HKV, DH)
    q = pkg.kv_append(cache, batch, x[:, HQ:HQ + HKV], x[:, HQ + HKV:], q=x[:, :HQ], norm_eps=EPS, rope_cos=cos, rope_sin=sin,
                      rope_order=pkg.ROPE_SPLIT)
    attn = pkg.paged_attention(q, cache, batch, causal_block=block, window=window, workspace=ws)
    q2, s2 = pkg.quantize_rows(attn.view(tokens.shape[0], -1))
    xa = lin(q2, s2, "w_out", "s_out", gate=L["gate0"], residual=tokens)
    x = xa
    if "w_ctrl_fc1" in L:
        q3, s3 = pkg.rms_norm_quantize_rows(xa, None, None, EPS)
        q4, s4 = pkg.quantize_rows(lin(q3, s3, "w_ctrl_fc1", "s_ctrl_fc1", bias=L.get("ctrl_cond"), act=pkg.ACT_SILU))
        x = lin(q4, s4, "w_ctrl_fc2", "s_ctrl_fc2", residual=xa)
    q5, s5 = pkg.rms_norm_quantize_rows(x, L["mod_scale1"], L["mod_bias1"], EPS, scale_is_mod=True)
    q6, s6 = pkg.quantize_rows(lin(q5, s5, "w_fc1", "s_fc1", act=pkg.ACT_SILU))
    return lin(q6, s6, "w_fc2", "s_fc2", gate=L["gate1"], residual=x), attn


@pytest.mark.parametrize("T,D,HQ,HKV,DH,HID,ctrl,use_slab,page,dtype,worlds,window",
                         [(96, 256, 4, 2, 64, 512, True, False, 16, "f16", 1, 0),
                          (33, 512, 4, 4, 128, 1024, False, True, 32, "bf16", 3, 50),
                          (1, 256, 4, 1, 64, 512, True, False, 64, "f16", 5, 0),
                          (512, 2048, 32, 16, 64, 8192, True, True, 64, "f16", 1, 0)])
def test_frames_equal_the_operator_composition(pkg, T, D, HQ, HKV, DH, HID, ctrl, use_slab, page, dtype, worlds, window):
    L, layout, cache, table, drv, g = setup(pkg, T, D, HQ, HKV, DH, HID, ctrl, use_slab, page, pr.DTYPES[dtype], worlds)
    other = pkg.PagedKVCache(cache.k_pages.clone(), cache.v_pages.clone())
    starts = torch.arange(worlds + 1, dtype=torch.int32, device=DEV) * T
    lens = torch.zeros(worlds, dtype=torch.int32, device=DEV)
    batch = pkg.PagedBatch(table, starts, lens, max_new_tokens=T)
    ws = pkg.make_attention_workspace(cache)
    packed = drv.pack(L)
    tokens = (torch.randn(worlds * T, D, generator=g) * 2).to(DEV)
    for step in range(4):
        lens += T
        pos, xy, inv_t = frame(worlds * T, DH, 32, 16, step)
        cos, sin = pkg.rope_tables(*[p.to(DEV) for p in pos], xy.to(DEV), inv_t.to(DEV), DH, 32, 16)
        nxt = drv.forward_paged(packed, tokens, cos, sin, cache, batch, causal_block=T, window=window, workspace=ws)
        want, _ = composition(pkg, L, layout, tokens, cos, sin, other, batch, HQ, HKV, DH, T, window, ws)
        torch.cuda.synchronize()
        assert pkg.poll_status() == 0
        assert torch.equal(nxt, want), step
        used = table.long()[:, :-(-int(lens[0]) // page)].flatten()
        for a, b in ((cache.k_pages, other.k_pages), (cache.v_pages, other.v_pages)):
            assert torch.equal(a[used].nan_to_num(7.0), b[used].nan_to_num(7.0))
        inplace = tokens.clone()  # tokens_next may be the tokens; the same step again writes the same places
        drv.forward_paged(packed, inplace, cos, sin, cache, batch, causal_block=T, window=window, out=inplace, workspace=ws)
        torch.cuda.synchronize()
        assert torch.equal(inplace, want)
        tokens = nxt
    drv.close()


def test_agrees_with_the_two_calls_around_an_attention_in_64_bits(pkg):
    """layer_qkv (its own norm and rotation, fp32) + attention over all frames in 64 bits + layer_after_attention, against
    forward_paged.  The roundings of queries, keys, values and attention to fp16 (2^-11 each, half a step) may move a code of
    the attention's quantizer by one step of 1 / 127 of its row's largest value; through the out linear and its gate that
    is a small share of the token stream's size.  Bounded: the difference of the streams in the 2-norm by 2^-6 of what the
    layer adds to the stream (four roundings of 2^-11 and a code step of 2^-7 with random signs stay below half of it)."""
    T, D, HQ, HKV, DH, HID = 96, 512, 8, 4, 64, 1024
    L, layout, cache, table, drv, g = setup(pkg, T, D, HQ, HKV, DH, HID, True, False, 32, torch.float16, 1)
    lens, starts = torch.zeros(1, dtype=torch.int32, device=DEV), torch.tensor([0, T], dtype=torch.int32, device=DEV)
    batch = pkg.PagedBatch(table, starts, lens)
    packed, keys, values = drv.pack(L), [], []
    for step in range(3):
        lens += T
        tokens = (torch.randn(T, D, generator=g) * 2).to(DEV)
        pos, xy, inv_t = frame(T, DH, 32, 16, step)
        cos, sin = pkg.rope_tables(*[p.to(DEV) for p in pos], xy.to(DEV), inv_t.to(DEV), DH, 32, 16)
        q, k, v = drv.qkv(packed, tokens, cos, sin)
        keys.append(k)
        values.append(v)
        kk, vv = (torch.cat(x, 1).double().repeat_interleave(HQ // HKV, 0) for x in (keys, values))
        w = torch.softmax(q.double() @ kk.transpose(1, 2) * DH ** -0.5, -1)
        attn = (w @ vv).permute(1, 0, 2).reshape(T, D).float().contiguous()
        want = drv.after_attention(packed, attn, tokens)
        got = drv.forward_paged(packed, tokens, cos, sin, cache, batch, causal_block=T)
        torch.cuda.synchronize()
        assert pkg.poll_status() == 0
        off = float((got - want).double().norm() / (want - tokens).double().norm())
        assert off <= 2.0 ** -6, (step, off)
    drv.close()


def test_refusals(pkg):
    T, D, HQ, HKV, DH, HID = 32, 256, 4, 2, 64, 512
    L, layout, cache, table, drv, g = setup(pkg, T, D, HQ, HKV, DH, HID, True, False, 16, torch.float16, 1)
    batch = pkg.PagedBatch(table, torch.tensor([0, T], dtype=torch.int32, device=DEV), torch.tensor([T], dtype=torch.int32, device=DEV))
    tokens = torch.zeros(T, D, device=DEV)
    cos = torch.ones(T, DH // 2, device=DEV)
    packed = drv.pack(L)
    wide = pkg.PagedKVCache(*(torch.zeros(4, HKV + 1, 16, DH, dtype=torch.float16, device=DEV) for _ in range(2)))
    with pytest.raises(pkg.W8A8Error, match="heads"):
        drv.forward_paged(packed, tokens, cos, cos, wide, batch)
    with pytest.raises(pkg.W8A8Error, match="table rows"):
        drv.forward_paged(packed, tokens, cos[:-1], cos[:-1], cache, batch)
    with pytest.raises(pkg.W8A8Error, match="context holds"):
        drv.forward_paged(packed, torch.zeros(T + 1, D, device=DEV), torch.ones(T + 1, DH // 2, device=DEV),
                          torch.ones(T + 1, DH // 2, device=DEV), cache, batch)
    with pytest.raises(pkg.W8A8Error, match="invalid layer_forward_paged"):
        drv.forward_paged(drv.pack({k: v for k, v in L.items() if k != "w_fc1"}), tokens, cos, cos, cache, batch)
    with pytest.raises(pkg.W8A8Error, match="controller branch"):
        drv.forward_paged(drv.pack({k: v for k, v in L.items() if k != "w_ctrl_fc2"}), tokens, cos, cos, cache, batch)
    with pytest.raises(pkg.W8A8Error, match="workspace"):
        drv.forward_paged(packed, tokens, cos, cos, cache, batch, workspace=torch.zeros(256, dtype=torch.uint8, device=DEV))
    drv.close()


def test_a_refused_layer_leaves_the_cache_alone(pkg):
    """What the attention would refuse is refused before keys and values are written."""
    T, D, HQ, HKV, DH, HID = 32, 256, 4, 2, 64, 512
    L, layout, cache, table, drv, g = setup(pkg, T, D, HQ, HKV, DH, HID, True, False, 16, torch.float16, 1)
    batch = pkg.PagedBatch(table, torch.tensor([0, T], dtype=torch.int32, device=DEV), torch.tensor([T], dtype=torch.int32, device=DEV))
    tokens, cos, packed = torch.ones(T, D, device=DEV), torch.ones(T, DH // 2, device=DEV), drv.pack(L)
    small = torch.zeros(256, dtype=torch.uint8, device=DEV)
    for kw, match in ((dict(causal_block=0, window=5), "window"), (dict(causal_block=-1), "causal_block"), (dict(workspace=small), "workspace")):
        with pytest.raises(pkg.W8A8Error, match=match):
            drv.forward_paged(packed, tokens, cos, cos, cache, batch, **kw)
    torch.cuda.synchronize()
    assert bool(cache.k_pages.isnan().all()) and bool(cache.v_pages.isnan().all())
    assert bool(drv.forward_paged(packed, tokens, cos, cos, cache, batch).isfinite().all())
    drv.close()
