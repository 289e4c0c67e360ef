"""Cases of the paged key / value cache: appending to it (per-head norm and rotation on the way) and attention of new
tokens over it, each with a plain form in elementary torch operations and the calls that a user of the library makes.

The cache is a pool of pages, [pages, kv_heads, page_tokens, d_head] as the kernels see it; the memory is ordered that way
("heads") or [pages, page_tokens, kv_heads, d_head] ("tokens").  A batch of sequences has a page table [seqs, pages of the
longest], the row at which each sequence's new tokens start (seqs + 1 entries) and each sequence's number of keys, the new
tokens among them.  New token i of a sequence with n new tokens and L keys stands at position L - n + i.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


# ------------------------------------------------------------------ cases
def _append(name, **kw):
    return dict({"name": name, "op": "append"}, **kw)


def _attend(name, **kw):
    return dict({"name": name, "op": "attend"}, **kw)


def listed():
    return [
        # one token of one sequence: a single user's decoding step, all latency
        _append("append_one_token", seqs=1, new=1, keys=777, heads=32, kv_heads=16, d_head=64, page=64, order="heads",
                x="f32", dtype="f16", rope="split", table="token", weights=False),
        # a frame of 512 tokens through the layer's own QKV linear (fp32 rows), the framework's rotation tables
        _append("append_frame", seqs=1, new=512, keys=8192, heads=32, kv_heads=16, d_head=64, page=64, order="heads",
                x="f32", dtype="f16", rope="split", table="token", weights=False),
        # a decoding step of many sequences of ragged length, small pages, norms with weights, a table by position
        _append("append_decode_batch", seqs=128, new=1, keys=8191, heads=32, kv_heads=8, d_head=128, page=16,
                order="tokens", x="bf16", dtype="bf16", rope="halves", table="position", weights=True),
        # 64 worlds x 2048 rows, the rows of the default benchmark
        _append("append_worlds", seqs=64, new=2048, keys=2048, heads=32, kv_heads=16, d_head=64, page=128,
                order="heads", x="f16", dtype="f16", rope="pairs", table="token", weights=False),
        # single user, short cache: latency
        _attend("attend_one_token", seqs=1, new=1, keys=777, heads=32, kv_heads=16, d_head=64, page=64, order="heads",
                dtype="f16", block=1, window=0),
        # decoding of a batch of ragged sequences: reads the cache once
        _attend("attend_decode_batch", seqs=64, new=1, keys=8191, heads=32, kv_heads=8, d_head=128, page=16,
                order="tokens", dtype="bf16", block=1, window=0),
        # decoding of one very long sequence: the key axis has to be split
        _attend("attend_decode_long", seqs=1, new=1, keys=131071, heads=32, kv_heads=8, d_head=128, page=64,
                order="heads", dtype="bf16", block=1, window=0),
        # a few tokens each (drafts to be verified), 16 heads to a key head
        _attend("attend_few_tokens", seqs=16, new=5, keys=4001, heads=32, kv_heads=2, d_head=128, page=32,
                order="heads", dtype="f16", block=1, window=0),
        # one frame of 512 tokens over 16 frames of cache and itself: the layer's own shape, causal by frames
        _attend("attend_frame", seqs=1, new=512, keys=8704, heads=32, kv_heads=16, d_head=64, page=64, order="heads",
                dtype="f16", block=512, window=0),
        # chunks of ragged prompts over what is cached, 7 heads to a key head
        _attend("attend_chunks", seqs=8, new=1000, keys=6007, heads=28, kv_heads=4, d_head=128, page=32,
                order="tokens", dtype="bf16", block=1, window=0),
        # a sliding window over long sequences, 3 heads to a key head
        _attend("attend_window", seqs=4, new=2048, keys=16001, heads=24, kv_heads=8, d_head=64, page=16, order="heads",
                dtype="f16", block=1, window=1000),
        # a whole prompt at once
        _attend("attend_prompt", seqs=1, new=8192, keys=8192, heads=32, kv_heads=8, d_head=128, page=128,
                order="heads", dtype="bf16", block=1, window=0),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    d_head = rng.choice([64, 128])
    group, kv_heads = rng.choice([(1, 12), (2, 16), (3, 6), (4, 5), (5, 4), (7, 4), (8, 4), (16, 2), (6, 1), (2, 3)])
    case = {"heads": group * kv_heads, "kv_heads": kv_heads, "d_head": d_head, "page": rng.choice([16, 32, 64, 128]),
            "order": rng.choice(["heads", "tokens"]), "dtype": rng.choice(["f16", "bf16"])}
    if rng.random() < 0.35:
        seqs = _spread(rng, 1, 128)
        new = _spread(rng, 1, max(1, min(2048, 100000 // seqs)))
        keys = new + rng.choice([0, 1, 1]) * _spread(rng, 1, 8000)
        return dict(case, op="append", seqs=seqs, new=new, keys=min(keys, max(new, 300000 // seqs)),
                    x=rng.choice(["f32", case["dtype"]]), rope=rng.choice(["none", "split", "halves", "pairs"]),
                    table=rng.choice(["token", "position"]), weights=rng.random() < 0.5)
    new = rng.choice([1, 1, _spread(rng, 2, 16), _spread(rng, 17, 4096)])
    scores = 2 ** 30  # heads x new tokens x keys of all sequences: half of the largest listed case
    seqs = min(_spread(rng, 1, 64), max(1, scores // (case["heads"] * new * max(new, 64))))
    keys = _spread(rng, max(new, 1), max(new, min(100000, scores // (case["heads"] * new * seqs), 400000 // seqs)))
    block = rng.choice([1, 1, 1, 0, _spread(rng, 2, 600)])
    return dict(case, op="attend", seqs=seqs, new=new, keys=keys, block=block,
                window=_spread(rng, 1, 5000) if block and rng.random() < 0.3 else 0)


def _lengths(case):
    """(new tokens, keys) of each sequence: the first has the most of both, the others between a half and all."""
    part = [1.0 - 0.5 * ((0.6180339887 * i) % 1.0) for i in range(case["seqs"])]
    new = [max(1, round(case["new"] * p)) for p in part]
    keys = [max(n, round(case["keys"] * p)) for n, p in zip(new, part)]
    return new, keys


def _visible(case):
    """For each sequence, (first key, one past the last key) of every new token, as two tensors."""
    found = []
    for n, keys in zip(*_lengths(case)):
        position = keys - n + torch.arange(n, dtype=torch.int64)
        low, high = torch.zeros_like(position), torch.full_like(position, keys)
        if case["block"]:
            end = (torch.div(position, case["block"], rounding_mode="floor") + 1) * case["block"]
            high = torch.minimum(high, end)
            if case["window"]:
                low = (end - case["window"]).clamp(min=0)
        found.append((low, torch.maximum(low, high)))
    return found


def work(case):
    tokens = sum(_lengths(case)[0])
    heads, kv_heads, d_head = case["heads"], case["kv_heads"], case["d_head"]
    if case["op"] == "append":
        numbers = tokens * (heads + 2 * kv_heads) * d_head
        read = numbers * (4 if case["x"] == "f32" else 2) + (0 if case["rope"] == "none" else tokens * d_head * 4)
        return {"bytes": read + numbers * 2, "flops": 8 * numbers}
    seen = _visible(case)
    pairs = sum(int((high - low).sum()) for low, high in seen)
    keys = sum(int(high.max() - low.min()) for low, high in seen)
    return {"bytes": 4 * d_head * (tokens * heads + keys * kv_heads), "flops": 4 * pairs * heads * d_head}


# ------------------------------------------------------------------ what a program has in hand
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    new, keys = _lengths(case)
    seqs, page, d_head = case["seqs"], case["page"], case["d_head"]
    kv_heads, heads, dtype = case["kv_heads"], case["heads"], DTYPES[case["dtype"]]
    tokens = sum(new)
    counts = [-(-n // page) for n in keys]
    pages = sum(counts)
    # a page table as an allocator leaves it: pages in any order, entries behind a sequence's last page unused (0)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(seqs, max(counts), dtype=torch.int32, device="cuda")
    filled = torch.arange(max(counts), device="cuda")[None, :] < torch.tensor(counts, device="cuda")[:, None]
    table[filled] = order
    shape = (pages, kv_heads, page, d_head) if case["order"] == "heads" else (pages, page, kv_heads, d_head)
    k_pages, v_pages = (torch.empty(shape, dtype=dtype, device="cuda") for _ in range(2))
    for pool in (k_pages, v_pages):
        step = max(1, 2 ** 26 // (page * kv_heads * d_head))
        for at in range(0, pages, step):  # in pieces: 32-bit random numbers of the whole pool would take twice its room
            pool[at:at + step] = randn(min(step, pages - at), *shape[1:]).to(dtype)
    if case["order"] == "tokens":
        k_pages, v_pages = k_pages.transpose(1, 2), v_pages.transpose(1, 2)
    starts = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    state = {"case": dict(case), "k_pages": k_pages, "v_pages": v_pages, "table": table, "starts": starts,
             "lens": torch.tensor(keys, dtype=torch.int32, device="cuda"), "most_new": max(new), "most_keys": max(keys)}
    if case["op"] == "attend":
        # normed queries with a gain for each head, as a model learns them: from nearly even to peaked weights
        gain = 1.0 + 3.0 * torch.rand(heads, 1, generator=g, device="cuda")
        q = randn(tokens, heads, d_head)
        state["q"] = (q * torch.rsqrt(q.square().mean(-1, keepdim=True)) * gain).to(dtype)
        state["out"] = torch.zeros_like(state["q"])
        return state
    # rows of a fused QKV linear, channels of unequal size
    x = randn(tokens, (heads + 2 * kv_heads) * d_head)
    state["x"] = (x * torch.exp(0.5 * randn(x.shape[1]))).to(DTYPES[case["x"]])
    state["q_out"] = torch.zeros(tokens, heads, d_head, dtype=dtype, device="cuda")
    if case["weights"]:
        state["q_weight"], state["k_weight"] = 1.0 + 0.1 * randn(d_head), 1.0 + 0.1 * randn(d_head)
    if case["rope"] != "none":
        where = torch.arange(max(keys), device="cuda")
        if case["table"] == "token":
            where = torch.cat([torch.arange(n - m, n) for m, n in zip(new, keys)]).cuda()
        inv = 10000.0 ** (-torch.arange(d_head // 2, dtype=torch.float64, device="cuda") / (d_head // 2))
        angle = where.double()[:, None] * inv
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _own_append(state) if state["case"]["op"] == "append" else _own_attend(state)
    return _plain_append(state) if state["case"]["op"] == "append" else _plain_attend(state)


def _package():
    import importlib.util
    import sys
    name = "worldmodel_cu_b200"  # the directory's name has a dot
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(name, "worldmodel.cu_b200/__init__.py")
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


def _handles(state):
    """The cache and batch objects that a program makes once for its buffers, and the attention's workspace."""
    if "cache" not in state:
        pkg = _package()
        state["cache"] = pkg.PagedKVCache(state["k_pages"], state["v_pages"])
        state["batch"] = pkg.PagedBatch(state["table"], state["starts"], state["lens"], max_new_tokens=state["most_new"])
        state["workspace"] = pkg.make_attention_workspace(state["cache"])
    return _package(), state["cache"], state["batch"]


def _own_append(state):
    case = state["case"]
    pkg, cache, batch = _handles(state)
    q, k, v = _heads_of(state["x"], case)
    order = {"none": None, "split": pkg.ROPE_SPLIT, "halves": pkg.ROPE_HALVES, "pairs": pkg.ROPE_PAIRS}[case["rope"]]
    pkg.kv_append(cache, batch, k, v, q=q, q_out=state["q_out"], norm_eps=EPS, q_weight=state.get("q_weight"),
                  k_weight=state.get("k_weight"), rope_cos=state.get("cos"), rope_sin=state.get("sin"),
                  rope_order=order, rope_by_position=case["table"] == "position")
    return {"q": state["q_out"], "k_pages": state["k_pages"], "v_pages": state["v_pages"]}


def _own_attend(state):
    case = state["case"]
    pkg, cache, batch = _handles(state)
    return pkg.paged_attention(state["q"], cache, batch, causal_block=case["block"], window=case["window"],
                               out=state["out"], workspace=state["workspace"])


def _heads_of(x, case):
    """Queries, keys and values [tokens, heads, d_head] in the rows of a fused QKV linear."""
    heads, kv_heads, d_head = case["heads"], case["kv_heads"], case["d_head"]
    parts = x.view(x.shape[0], heads + 2 * kv_heads, d_head)
    return parts[:, :heads], parts[:, heads:heads + kv_heads], parts[:, heads + kv_heads:]


def _places(state):
    """Sequence, index within it and position of every new token."""
    starts, lens = state["starts"].long(), state["lens"].long()
    tokens = torch.arange((state["x"] if "x" in state else state["q"]).shape[0], device="cuda")
    seq = torch.searchsorted(starts[1:], tokens, right=True)
    index = tokens - starts[seq]
    return seq, index, lens[seq] - (starts[seq + 1] - starts[seq]) + index


def _plain_append(state):
    case = state["case"]
    seq, _, position = _places(state)
    q, k, v = (part.float() for part in _heads_of(state["x"], case))
    turned = []
    for part, weight in ((q, state.get("q_weight")), (k, state.get("k_weight"))):
        part = part * torch.rsqrt(part.square().mean(-1, keepdim=True) + EPS)
        if weight is not None:
            part = part * weight
        if case["rope"] != "none":
            row = position if case["table"] == "position" else torch.arange(position.shape[0], device="cuda")
            cos, sin = state["cos"][row][:, None, :], state["sin"][row][:, None, :]
            half = part.shape[-1] // 2
            if case["rope"] == "halves":
                a, b = part[..., :half], part[..., half:]
            else:
                a, b = part[..., 0::2], part[..., 1::2]
            a, b = a * cos - b * sin, b * cos + a * sin
            part = torch.stack((a, b), -1).flatten(-2) if case["rope"] == "pairs" else torch.cat((a, b), -1)
        turned.append(part)
    page = state["table"].long()[seq, position // case["page"]]
    slot = position % case["page"]
    state["k_pages"][page, :, slot] = turned[1].to(state["k_pages"].dtype)
    state["v_pages"][page, :, slot] = v.to(state["v_pages"].dtype)
    state["q_out"].copy_(turned[0])
    return {"q": state["q_out"], "k_pages": state["k_pages"], "v_pages": state["v_pages"]}


def _plain_attend(state):
    case = state["case"]
    seqs, new, keys = case["seqs"], state["most_new"], state["most_keys"]
    kv_heads, d_head = case["kv_heads"], case["d_head"]
    group = case["heads"] // kv_heads
    starts, lens = state["starts"].long(), state["lens"].long()
    seq, index, _ = _places(state)
    used = state["table"][:, :-(-keys // case["page"])].long()
    k, v = (pool[used].transpose(1, 2).reshape(seqs, kv_heads, -1, d_head)[:, :, :keys].float()
            for pool in (state["k_pages"], state["v_pages"]))
    count = starts[1:] - starts[:-1]
    lane = torch.arange(new, device="cuda")
    padded = (starts[:-1, None] + lane).clamp(max=state["q"].shape[0] - 1)
    q = state["q"][padded].view(seqs, new, kv_heads, group, d_head).permute(0, 2, 3, 1, 4).float()
    scores = q.reshape(seqs, kv_heads, group * new, d_head) @ k.transpose(-1, -2)
    scores = scores.mul_(1.0 / math.sqrt(d_head)).view(seqs, kv_heads, group, new, keys)
    position = (lens - count)[:, None] + lane
    key = torch.arange(keys, device="cuda")
    hidden = (key >= lens[:, None, None]).expand(seqs, new, keys)
    if case["block"]:
        end = (position // case["block"] + 1) * case["block"]
        hidden = hidden | (key >= end[..., None])
        if case["window"]:
            hidden = hidden | (key < end[..., None] - case["window"])
    hidden = hidden[:, None, None]
    scores.masked_fill_(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    out = scores.view(seqs, kv_heads, group * new, keys) @ v
    out = out.view(seqs, kv_heads, group, new, d_head) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs, new, case["heads"], d_head)
    state["out"].copy_(out[seq, index])
    return state["out"]


# ------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    new, keys = _lengths(case)
    if case["op"] == "append":
        return _exact_append(case, state, new, keys)
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    group, first = case["heads"] // case["kv_heads"], 0
    for s, (low, high) in enumerate(_visible(case)):
        n, most = new[s], keys[s]
        where = torch.arange(most, device="cuda")
        page, slot = state["table"][s].long()[where // case["page"]], where % case["page"]
        seen = (where >= low.cuda()[:, None]) & (where < high.cuda()[:, None])
        for h in range(case["heads"]):
            k = state["k_pages"][page, h // group, slot].double()
            v = state["v_pages"][page, h // group, slot].double()
            score = state["q"][first:first + n, h].double() @ k.T / math.sqrt(case["d_head"])
            weight = torch.softmax(score.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
            out[first:first + n, h] = weight @ v
        first += n
    return out


def _exact_append(case, state, new, keys):
    k_pages, v_pages = state["k_pages"].double(), state["v_pages"].double()
    x = state["x"].double().view(sum(new), -1, case["d_head"])
    heads, kv_heads, half = case["heads"], case["kv_heads"], case["d_head"] // 2
    position = torch.cat([torch.arange(n - m, n) for m, n in zip(new, keys)]).cuda()
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
    both = x[:, :heads + kv_heads]
    both = both / torch.sqrt((both * both).sum(-1, keepdim=True) / case["d_head"] + EPS)
    if case["weights"]:
        both = torch.cat((both[:, :heads] * state["q_weight"].double(), both[:, heads:] * state["k_weight"].double()), 1)
    if case["rope"] != "none":
        at = position if case["table"] == "position" else torch.arange(len(position), device="cuda")
        turn = torch.complex(state["cos"].double()[at], state["sin"].double()[at])[:, None]
        pair = both.unflatten(-1, (2, half)).transpose(-1, -2) if case["rope"] == "halves" else both.unflatten(-1, (half, 2))
        pair = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        both = pair.flatten(-2) if case["rope"] == "pairs" else pair.transpose(-1, -2).flatten(-2)
    page, slot = state["table"].long()[seq, position // case["page"]], position % case["page"]
    k_pages[page, :, slot] = both[:, heads:]
    v_pages[page, :, slot] = x[:, heads + kv_heads:]
    return {"q": both[:, :heads], "k_pages": k_pages, "v_pages": v_pages}
