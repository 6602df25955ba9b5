"""Performance cases of attention with a window and first tokens that stay, and of
caches in 8 bits with a scale for each block of tokens and head (sym_amd.attention).

In training, `window_attention` and its backward over packed sequences. In
serving, `block_append`, which quantizes a step's keys and values into the
cache and keeps each block's scale, and `tree_attention` over such a cache, or
over a 16-bit one, whole or with a window. A case is one of these calls (in
training with its backward).

`run` computes them in plain 32-bit torch operations, or through the package
where `own` is set. Lengths are part of a case (they follow from its values);
the seed makes the tensors, the page order and the trees.
"""
import math
import random
import zlib

import torch

own = False

WORD = 64           # rows of a tree that one mask word holds
ROWS = 128          # query rows that the plain training form takes at a time
LEAST = 2.0 ** -126  # of a block's scale
_contexts = {}


def _device():
    return torch.device("cuda", 0)


def _attention():
    """The package and one retained context, as a program keeps them."""
    if not _contexts:
        from sym_amd import attention, pyreloc
        _contexts["attention"], _contexts["context"] = attention, pyreloc.Context(0)
    return _contexts["attention"], _contexts["context"]


def listed():
    return [
        # a training micro-batch of packed documents, forward alone (evaluation)
        dict(name="window 8x4096", op="window", sequences=8, longest=4096, window=1024, sinks=4, heads=32, kv_heads=8, dim=128,
             dtype="bfloat16", back=False),
        # a few short documents, odd in every size: latency
        dict(name="window odd 5x333", op="window", sequences=5, longest=333, window=100, sinks=1, heads=12, kv_heads=4, dim=80,
             dtype="float16", back=False),
        # the training step of the first case: forward and backward
        dict(name="window step 8x4096", op="window", sequences=8, longest=4096, window=1024, sinks=4, heads=32, kv_heads=8,
             dim=128, dtype="bfloat16", back=True),
        # one long document with a wide window, as many key heads as query heads
        dict(name="window step 1x16384", op="window", sequences=1, longest=16384, window=4096, sinks=16, heads=16, kv_heads=16,
             dim=64, dtype="float16", back=True),
        # a decoding step's tokens into blocks that already hold some: latency
        dict(name="append 64x1", op="append", requests=64, longest=60, fresh=1, kv_heads=8, dim=128, dtype="bfloat16", page=64,
             block=64, order="slots"),
        # chunks of a few prompts into a head-major cache of large pages
        dict(name="append 4x4096 head-major", op="append", requests=4, longest=1000, fresh=4096, kv_heads=8, dim=128,
             dtype="bfloat16", page=256, block=32, order="heads"),
        # odd lengths and an odd head size
        dict(name="append odd 13x77", op="append", requests=13, longest=301, fresh=77, kv_heads=5, dim=80, dtype="float16",
             page=48, block=16, order="slots"),
        # one request decodes alone over blocks: latency
        dict(name="attend blocks 1x1 over 1000", op="attend", requests=1, longest=1000, fresh=1, tree=False, heads=32,
             kv_heads=8, dim=128, dtype="bfloat16", cache="blocks", page=64, block=64, order="slots", window=0, sinks=0),
        # a full batch decodes over blocks, all of its context
        dict(name="attend blocks 64x1 over 8192", op="attend", requests=64, longest=8192, fresh=1, tree=False, heads=32,
             kv_heads=8, dim=128, dtype="bfloat16", cache="blocks", page=64, block=64, order="slots", window=0, sinks=0),
        # drafted trees over blocks
        dict(name="attend blocks tree 8x48 over 8192", op="attend", requests=8, longest=8192, fresh=48, tree=True, heads=32,
             kv_heads=8, dim=128, dtype="float16", cache="blocks", page=128, block=32, order="slots", window=0, sinks=0),
        # a batch decodes with a window over long contexts in 16 bits
        dict(name="attend window 64x1 over 32768", op="attend", requests=64, longest=32768, fresh=1, tree=False, heads=32,
             kv_heads=8, dim=128, dtype="bfloat16", cache="bfloat16", page=16, block=16, order="slots", window=2048, sinks=4),
        # chunks of long prompts with a window over blocks
        dict(name="attend window chunk 4x512 blocks", op="attend", requests=4, longest=16384, fresh=512, tree=False, heads=32,
             kv_heads=8, dim=128, dtype="bfloat16", cache="blocks", page=64, block=64, order="heads", window=2048, sinks=4),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["window", "window", "append", "attend", "attend"])
    dtype = rng.choice(["bfloat16", "float16"])
    if op == "window":
        kv_heads = rng.choice([1, 2, 4, 8, 16])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 8] if kv_heads < 8 else [1, 4] if kv_heads < 16 else [1])
        dim = rng.choice([64, 80, 96, 128, 128])
        sequences = _spread(rng, 1, 16)
        back = rng.random() < 0.5
        longest = _spread(rng, 1, 32768 // sequences)
        # no more pairs of tokens, over the heads, than the largest listed case has
        most = 32768 * 1024 * 32 * 128 * 6 // (sequences * longest * heads * dim * (7 if back else 2))
        return dict(op=op, sequences=sequences, longest=longest, window=_spread(rng, 1, max(2, min(longest, most // 2))),
                    sinks=rng.choice([0, 1, 4, 4, 17, 64]), heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, back=back)
    kv_heads = rng.choice([1, 2, 5, 8, 32])
    dim = rng.choice([64, 80, 128, 128, 256])
    block = rng.choice([16, 32, 64, 128])
    page = block * rng.choice([1, 1, 2, 3])
    order = rng.choice(["slots", "heads"])
    if op == "append":
        requests = _spread(rng, 1, 256)
        most = 4 * 5096 * 8 * 128 // (requests * kv_heads * dim)
        fresh = _spread(rng, 1, max(1, min(4096, most // 2)))
        return dict(op=op, requests=requests, longest=rng.randint(0, max(1, min(1000, most // 2))), fresh=fresh,
                    kv_heads=kv_heads, dim=dim, dtype=dtype, page=page, block=block, order=order)
    heads = kv_heads * (1 if kv_heads == 32 else rng.choice([1, 3, 4, 8]))
    requests = _spread(rng, 1, 64)
    tree = rng.random() < 0.4
    fresh = _spread(rng, 1, WORD if tree else 256)
    cache = rng.choice([dtype, "blocks", "blocks"])
    # no more tokens than the largest listed cases hold, nor more scores in the plain form
    most = min(65536, 2 ** 30 // (requests * kv_heads * dim * (1 if cache == "blocks" else 2)), 2 ** 29 // (requests * heads * fresh))
    longest = _spread(rng, 1, max(2, most))
    window = rng.choice([0, _spread(rng, WORD if tree else 1, 8192)])
    return dict(op=op, requests=requests, longest=longest, fresh=fresh, tree=tree, heads=heads, kv_heads=kv_heads, dim=dim,
                dtype=dtype, cache=cache, page=page, block=block, order=order, window=window,
                sinks=rng.choice([0, 1, 4, 33]) if window else 0)


def _case_rng(case):
    key = repr(sorted((k, v) for k, v in case.items() if k not in ("name", "back")))
    return random.Random(zlib.crc32(key.encode()))


def _sequences(case):
    """Lengths of packed sequences: ragged where there are several, the longest as the case says."""
    rng, n, longest = _case_rng(case), case["sequences"], case["longest"]
    lengths = [rng.randint((longest + 1) // 2, longest) for _ in range(n)]
    lengths[rng.randrange(n)] = longest
    return lengths


def _lengths(case):
    """(cached, fresh) of every request: ragged where there are several, the longest as the case says."""
    rng, n, longest, fresh = _case_rng(case), case["requests"], case["longest"], case["fresh"]
    cached = [rng.randint(longest // 2, longest) for _ in range(n)]
    new = [rng.randint((fresh + 1) // 2, fresh) for _ in range(n)]
    cached[rng.randrange(n)], new[rng.randrange(n)] = longest, fresh
    return cached, new


def _pages(n, page):
    return -(-n // page)


def _words(rng, n):
    """A drafted tree, each token following one of the last few before it or the context: its tokens' ancestors,
    themselves among them, as mask words."""
    rows = []
    for j in range(n):
        p = rng.randint(max(-1, j - 6), j - 1)
        rows.append((1 << j) | (rows[p] if p >= 0 else 0))
    return [r - (1 << WORD) if r >> (WORD - 1) else r for r in rows]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=_device())


def _starts(lengths):
    total = [0]
    for n in lengths:
        total.append(total[-1] + n)
    return _ints(total)


def _order(case, gen, pages, codes):
    """A cache of `pages` pages, [pages, page, kv_heads, dim], slot-major or (viewed) head-major in memory."""
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    shape = (pages, page, heads, dim) if case["order"] == "slots" else (pages, heads, page, dim)
    if codes:
        t = torch.randint(-100, 101, shape, generator=gen, device=_device(), dtype=torch.int8)
    else:
        t = torch.randn(shape, generator=gen, device=_device(), dtype=getattr(torch, case["dtype"]))
    return t if case["order"] == "slots" else t.transpose(1, 2)


def _page_table(gen, lengths, page):
    """A table of pages in no order, -1 past each request's own, and how many pages the pool has."""
    need = [_pages(n, page) for n in lengths]
    pool = sum(need) + 3
    ids = torch.randperm(pool, generator=gen, device=_device(), dtype=torch.int64).to(torch.int32)
    counts = torch.tensor(need, device=_device())
    at = torch.arange(max(need), device=_device())[None, :]
    first = (counts.cumsum(0) - counts)[:, None]
    table = torch.where(at < counts[:, None], ids[(first + at).clamp(max=pool - 1)], -1)
    return table.to(torch.int32).contiguous(), pool


def _scales(case, gen, pages):
    shape = (pages, case["page"] // case["block"], case["kv_heads"])
    return torch.rand(shape, generator=gen, device=_device()) * 0.02 + 0.01


def prepare(case, seed):
    c, s = case, {"case": case}
    gen = torch.Generator(device=_device()).manual_seed(seed)
    heads, kv, dim, dtype = c.get("heads"), c["kv_heads"], c["dim"], getattr(torch, c["dtype"])

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=_device(), dtype=dtype)
    if c["op"] == "window":
        lengths = _sequences(c)
        n = sum(lengths)
        s["starts"] = _starts(lengths)
        # queries, keys and values as views of the fused projection
        fused = randn(n, (heads + 2 * kv) * dim)
        s["q"] = fused[:, :heads * dim].unflatten(1, (heads, dim))
        s["k"] = fused[:, heads * dim:(heads + kv) * dim].unflatten(1, (kv, dim))
        s["v"] = fused[:, (heads + kv) * dim:].unflatten(1, (kv, dim))
        if c["back"]:
            s["do"] = randn(n, heads, dim)
        # where the plain form's pieces of ROWS rows begin: sequence by sequence
        s["piece_seq"] = _ints([b for b, m in enumerate(lengths) for _ in range(0, m, ROWS)])
        s["piece_row"] = _ints([r for m in lengths for r in range(0, m, ROWS)])
        s["reach"] = min(c["window"], max(lengths))
        return s
    cached, fresh = _lengths(c)
    rows, lengths = sum(fresh), [a + b for a, b in zip(cached, fresh)]
    s.update(cached=_ints(cached), starts=_starts(fresh))
    s["table"], pool = _page_table(gen, lengths, c["page"])
    codes = c["op"] == "append" or c["cache"] == "blocks"
    s["cache_k"], s["cache_v"] = _order(c, gen, pool, codes), _order(c, gen, pool, codes)
    s["k_scale"], s["v_scale"] = (_scales(c, gen, pool), _scales(c, gen, pool)) if codes else (None, None)
    if c["op"] == "append":
        # tokens of several sizes: some of them make their block's scale grow
        size = torch.exp(0.5 * torch.randn((rows, kv, 1), generator=gen, device=_device()))
        s["k"], s["v"] = (randn(rows, kv, dim) * size).to(dtype), randn(rows, kv, dim)
        return s
    s["q"] = randn(rows, heads, dim)
    rng = random.Random(seed)
    s["mask"] = torch.tensor([w for n in fresh for w in _words(rng, n)], device=_device())[:, None] if c["tree"] else None
    s["scale"] = dim ** -0.5
    s["most_rows"], s["most_tokens"] = max(fresh), max(lengths)
    return s


# ------------------------------------------------------------- plain forms

def _plain_window(s):
    """Attention of pieces of ROWS rows, each over the first tokens and the reach of its rows' windows; with
    gradients where the case has them."""
    c = s["case"]
    heads, kv, dim, sinks, reach = c["heads"], c["kv_heads"], c["dim"], c["sinks"], s["reach"]
    group, scale = heads // kv, dim ** -0.5
    starts = s["starts"].long()
    begin, n = starts[:-1][s["piece_seq"].long()][:, None], (starts[1:] - starts[:-1])[s["piece_seq"].long()][:, None]
    row0 = s["piece_row"].long()[:, None]
    at = torch.arange(ROWS, device=starts.device)[None, :] + row0  # places in the sequence
    real = at < n
    first = torch.arange(sinks, device=starts.device)[None, :].expand(row0.shape[0], sinks)
    near = torch.arange(ROWS + reach - 1, device=starts.device)[None, :] + row0 - (reach - 1)
    x = torch.cat([first, near], 1)  # tokens that some row of the piece may see
    back = at[:, :, None] - x[:, None, :]
    see = (back >= 0) & (x >= 0)[:, None, :] & real[:, :, None]
    see = see & torch.cat([back[:, :, :sinks] >= reach, back[:, :, sinks:] < reach], 2)
    rows, tokens = (begin + at.clamp(max=c["longest"])).clamp(max=s["q"].shape[0] - 1), begin + x.clamp(min=0)
    tokens = tokens.clamp(max=s["q"].shape[0] - 1)

    def take_rows(t):  # [pieces, kv, group * ROWS, dim]
        return t.float()[rows].unflatten(2, (kv, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)

    def give_rows(t):  # and back, [rows, heads, dim]
        return t.unflatten(2, (group, ROWS)).permute(0, 3, 1, 2, 4).flatten(2, 3)[real].to(s["q"].dtype)
    q, k, v = take_rows(s["q"]), s["k"].float()[tokens].transpose(1, 2), s["v"].float()[tokens].transpose(1, 2)
    hide = ~see[:, None, None]
    p = ((q @ k.transpose(2, 3)) * scale).unflatten(2, (group, ROWS)).masked_fill_(hide, -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True).clamp(min=-1e30))
    p = (p / p.sum(-1, keepdim=True).clamp(min=1e-30)).flatten(2, 3)
    o = p @ v
    if not c["back"]:
        return give_rows(o)
    do = take_rows(s["do"])
    ds = (do @ v.transpose(2, 3) - (do * o).sum(-1, keepdim=True)) * p * scale
    # a row outside its sequence repeats another: it sees nothing, so its weights are zero
    dk, dv = ds.transpose(2, 3) @ q, p.transpose(2, 3) @ do
    out = [give_rows(o), give_rows(ds @ k)]
    for g in (dk, dv):
        whole = torch.zeros(s["k"].shape, device=g.device)
        whole.index_add_(0, tokens.flatten(), g.transpose(1, 2).flatten(0, 1))
        out.append(whole.to(s["k"].dtype))
    return out


def _values(codes, scale, like, block):
    """What a cache's codes stand for, in the type of the operands."""
    out = torch.empty(codes.shape, dtype=like.dtype, device=codes.device)
    torch.mul(codes.unflatten(1, (-1, block)), scale[:, :, None, :, None], out=out.unflatten(1, (-1, block)))
    return out


def _updated(s):
    block = s["case"]["block"]
    return [_values(s["cache_k"], s["k_scale"], s["k"], block), _values(s["cache_v"], s["v_scale"], s["v"], block),
            s["k_scale"], s["v_scale"]]


def _plain_append(s):
    c, table = s["case"], s["table"].long()
    page, block = c["page"], c["block"]
    cached, starts = s["cached"].long(), s["starts"].long()
    fresh = starts[1:] - starts[:-1]
    row = torch.arange(s["k"].shape[0], device=table.device)
    req = torch.searchsorted(starts, row, right=True) - 1
    x = cached[req] + row - starts[req]
    ids, off = table[req, x // page], x % page
    # the blocks that the step touches, request by request
    count = torch.where(fresh > 0, (cached + fresh - 1) // block - cached // block + 1, 0)
    base = count.cumsum(0) - count
    mine = base[req] + x // block - cached[req] // block
    # tokens that are there already, in the first of them
    old = torch.arange(block, device=table.device)[None, :]
    have = (cached % block)[:, None]
    place = (cached - cached % block)[:, None] + old
    there = (old < have) & (fresh > 0)[:, None]
    old_ids = torch.where(there, table.gather(1, (place // page).clamp(max=table.shape[1] - 1)), 0)
    total = s["k"].shape[0] + cached.numel()  # at least as many as there are blocks
    for name in "kv":  # keys, then values
        cache, scale, new = s["cache_" + name], s[name + "_scale"], s[name].float()
        kv, most = new.shape[1], new.abs().amax(-1)
        most = torch.zeros((total, kv), device=new.device).index_reduce_(0, mine, most, "amax")
        held = scale[old_ids[:, 0], (place[:, 0] % page) // block]
        before = torch.zeros((total, kv), device=new.device)
        before.index_reduce_(0, base.clamp(max=total - 1), torch.where(there[:, :1], held, 0.0), "amax")
        now = torch.maximum(most * (1.0 / 127.0), before).clamp(min=LEAST)
        codes = torch.round(new * (1.0 / now)[mine][:, :, None]).clamp(-128, 127).to(torch.int8)
        shrink = held * (1.0 / now)[base.clamp(max=total - 1)]
        kept = cache[old_ids, place % page]
        kept = torch.where(there[:, :, None, None], torch.round(kept.float() * shrink[:, None, :, None]).to(torch.int8), kept)
        cache[old_ids[there], (place % page)[there]] = kept[there]
        cache[ids, off] = codes
        scale[ids, off // block] = now[mine]
    return _updated(s)


def _plain_attend(s):
    c, q = s["case"], s["q"]
    heads, kv, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    group, rows, tokens = heads // kv, s["most_rows"], s["most_tokens"]
    cached, starts, table = s["cached"].long(), s["starts"].long(), s["table"].long()
    window, sinks = c["window"] or tokens, c["sinks"]
    # the tokens that a request's rows may see: the first ones, and those from its first row's window on
    low = (cached - (window - 1)).clamp(min=sinks)[:, None]
    near = low + torch.arange(min(tokens, window + rows), device=q.device)[None, :]
    x = torch.cat([torch.arange(sinks, device=q.device)[None, :].expand(low.shape[0], sinks), near], 1)
    ids = table.gather(1, (x // page).clamp(max=table.shape[1] - 1)).clamp(min=0)
    k, v = s["cache_k"][ids, x % page].float(), s["cache_v"][ids, x % page].float()
    if s["k_scale"] is not None:
        at = (x % page) // c["block"]
        k, v = k * s["k_scale"][ids, at][..., None], v * s["v_scale"][ids, at][..., None]
    k, v = k.transpose(1, 2), v.transpose(1, 2)  # [B, kv, tokens, dim]
    j = torch.arange(rows, device=q.device)
    fresh = starts[1:] - starts[:-1]
    at = (starts[:-1, None] + j[None, :]).clamp(max=q.shape[0] - 1)
    w = q.float()[at].unflatten(2, (kv, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, kv, group * rows, dim]
    d = (x - cached[:, None])[:, None, :]  # the token's place among the fresh ones
    depth = j[None, :, None]
    if s["mask"] is not None:
        words = s["mask"][at]
        bits = (words >> torch.arange(WORD, device=q.device)) & 1
        depth = bits.sum(-1, keepdim=True) - 1
        see = (d < 0) | ((d < WORD) & (((words >> d.clamp(0, WORD - 1)) & 1) > 0))
        see = see & ((d >= 0) | (x[:, None, :] < sinks) | (depth - d < window))
    else:
        see = (d <= depth) & ((x[:, None, :] < sinks) | (depth - d < window))
    see = (see & (d < fresh[:, None, None]) & (j[None, :] < fresh[:, None])[:, :, None])[:, None, None]
    scores = ((w @ k.transpose(2, 3)) * s["scale"]).unflatten(2, (group, rows)).masked_fill(~see, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = (p.flatten(2, 3) @ v).unflatten(2, (group, rows)).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [B, rows, heads, dim]
    row = torch.arange(q.shape[0], device=q.device)
    req = torch.searchsorted(starts, row, right=True) - 1
    return o[req, row - starts[req]].to(q.dtype)


def run(s):
    c = s["case"]
    if own:
        A, ctx = _attention()
        if c["op"] == "window":
            see = dict(window=c["window"], sinks=c["sinks"])
            if not c["back"]:
                return A.window_attention(ctx, s["q"], s["k"], s["v"], s["starts"], **see)
            q, k, v = (s[x].detach().requires_grad_() for x in "qkv")
            o = A.window_attention(ctx, q, k, v, s["starts"], **see)
            return [o.detach(), *torch.autograd.grad(o, (q, k, v), s["do"])]
        if c["op"] == "append":
            A.block_append(ctx, s["k"], s["v"], s["cache_k"], s["cache_v"], s["k_scale"], s["v_scale"], s["table"], s["cached"],
                           s["starts"])
            return _updated(s)
        return A.tree_attention(ctx, s["q"], s["cache_k"], s["cache_v"], s["table"], s["cached"], s["starts"], mask=s["mask"],
                                scale=s["scale"], k_scale=s["k_scale"], v_scale=s["v_scale"], window=c["window"] or None,
                                sinks=c["sinks"])
    if c["op"] == "window":
        return _plain_window(s)
    return _plain_append(s) if c["op"] == "append" else _plain_attend(s)


def _pairs(n, window, sinks):
    """Pairs of a row and a token that it sees, in a sequence of n."""
    w = min(window, n)
    near = w * (w + 1) // 2 + (n - w) * w
    stay = sum(max(0, n - window - x) for x in range(min(sinks, n)))
    return near + stay


def work(case):
    c = case
    kv, dim = c["kv_heads"], c["dim"]
    if c["op"] == "window":
        lengths = _sequences(c)
        n, pairs = sum(lengths), sum(_pairs(m, c["window"], c["sinks"]) for m in lengths)
        rows, tokens = n * c["heads"] * dim * 2, 2 * n * kv * dim * 2
        # queries, keys, values and the result; its gradient, and those of the operands
        return {"bytes": (2 * rows + tokens) * (2 if c["back"] else 1), "flops": (14 if c["back"] else 4) * pairs * c["heads"] * dim}
    cached, fresh = _lengths(c)
    if c["op"] == "append":
        rows, cells = sum(fresh), 2 * kv * dim
        touched = sum(_pages(a + b, c["block"]) - a // c["block"] for a, b in zip(cached, fresh))
        # each element read in 16 bits and written in 8, each scale written; then the values of all pages read back, in 16
        pages = sum(_pages(a + b, c["page"]) for a, b in zip(cached, fresh)) + 3
        return {"bytes": rows * cells * 3 + touched * 2 * kv * 4 + pages * c["page"] * cells * 3, "flops": 4 * rows * cells}
    window, sinks, width = c["window"] or 1 << 40, c["sinks"], 2
    tokens = blocks = scores = 0
    for a, b in zip(cached, fresh):
        low = max(0, a - window + 1)
        seen = a + b - low + min(sinks, low)
        tokens += seen
        blocks += _pages(seen, c["block"])
        scores += sum(min(a + j + 1, window) + min(sinks, max(0, a + j + 1 - window)) for j in range(b))
    cell = 1 if c["cache"] == "blocks" else width
    more = blocks * 2 * kv * 4 if c["cache"] == "blocks" else 0
    return {"bytes": 2 * tokens * kv * dim * cell + more + 2 * sum(fresh) * c["heads"] * dim * width,
            "flops": 4 * scores * c["heads"] * dim}


# ---------------------------------------------- the definitions in 64 bits

def _exact_window(c, s):
    leaves = [s[x].double().requires_grad_(c["back"]) for x in "qkv"]
    group, starts, outs = c["heads"] // c["kv_heads"], s["starts"].tolist(), []
    grads = [torch.zeros_like(t) for t in leaves]
    with torch.set_grad_enabled(c["back"]):
        for a, b in zip(starts, starts[1:]):
            p = torch.arange(b - a, device=_device())
            see = (p[None, :] <= p[:, None]) & ((p[None, :] < c["sinks"]) | (p[:, None] - p[None, :] < c["window"]))
            for h in range(c["heads"]):
                q, k, v = leaves[0][a:b, h], leaves[1][a:b, h // group], leaves[2][a:b, h // group]
                scores = torch.where(see, q @ k.T * c["dim"] ** -0.5, -math.inf)
                o = torch.softmax(scores, -1) @ v
                outs.append((a, b, h, o.detach()))
                if c["back"]:
                    part = torch.autograd.grad(o, (q, k, v), s["do"][a:b, h].double())
                    for g, d, head in zip(grads, part, (h, h // group, h // group)):
                        g[a:b, head] += d
    whole = torch.zeros_like(leaves[0]).detach()
    for a, b, h, o in outs:
        whole[a:b, h] = o
    return [whole, *grads] if c["back"] else whole


def _exact_append(c, s):
    out, scales = [], []
    cached, starts, table = s["cached"].tolist(), s["starts"].tolist(), s["table"].tolist()
    page, block = c["page"], c["block"]
    for name in "kv":
        codes, scale, new = s["cache_" + name].double(), s[name + "_scale"].double(), s[name].double()
        for b, have in enumerate(cached):
            x, end = have, have + starts[b + 1] - starts[b]
            while x < end:
                first = x - x % block
                stop = min(first + block, end)
                at, off = table[b][first // page], first % page
                rows = new[starts[b] + x - have:starts[b] + stop - have]
                now = rows.abs().amax((0, 2)) / 127
                if x > first:
                    now = torch.maximum(now, scale[at, off // block])
                    part = codes[at, off:off + x - first]
                    codes[at, off:off + x - first] = torch.round(part * (scale[at, off // block] / now)[None, :, None])
                codes[at, off + x - first:off + stop - first] = torch.round(rows / now[None, :, None]).clamp(-128, 127)
                scale[at, off // block] = now
                x = stop
        out.append((codes.unflatten(1, (-1, block)) * scale[:, :, None, :, None]).flatten(1, 2))
        scales.append(scale)
    return out + scales


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] == "window":
        return _exact_window(c, s)
    if c["op"] == "append":
        return _exact_append(c, s)
    q, outs = s["q"].double(), []
    starts, cached, table = s["starts"].tolist(), s["cached"].tolist(), s["table"].long()
    group, window = c["heads"] // c["kv_heads"], c["window"] or 1 << 40
    for b in range(c["requests"]):
        r0, r1 = starts[b], starts[b + 1]
        n = cached[b] + r1 - r0
        ids = table[b, :_pages(n, c["page"])]
        k, v = s["cache_k"][ids].double(), s["cache_v"][ids].double()
        if s["k_scale"] is not None:
            k, v = (t * z[ids].double().repeat_interleave(c["block"], 1)[..., None] for t, z in ((k, s["k_scale"]), (v, s["v_scale"])))
        k, v = k.flatten(0, 1)[:n], v.flatten(0, 1)[:n]
        x = torch.arange(n, device=q.device)
        see = torch.zeros((r1 - r0, n), dtype=torch.bool, device=q.device)
        for j in range(r1 - r0):
            if s["mask"] is None:
                see[j] = x <= cached[b] + j
                at = cached[b] + j
            else:
                word = int(s["mask"][r0 + j, 0]) & ((1 << WORD) - 1)
                see[j, :cached[b]] = True
                see[j, cached[b]:] = torch.tensor([bool(word >> i & 1) for i in range(r1 - r0)], device=q.device)
                at = cached[b] + bin(word).count("1") - 1
            see[j] &= (x < c["sinks"]) | (at - x < window) | ((x >= cached[b]) & (s["mask"] is not None))
        heads = []
        for h in range(c["heads"]):
            a = (q[r0:r1, h] @ k[:, h // group].T * s["scale"]).masked_fill(~see, -math.inf)
            heads.append(torch.softmax(a, -1) @ v[:, h // group])
        outs.append(torch.stack(heads, 1))
    return torch.cat(outs)
