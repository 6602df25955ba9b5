"""Performance cases of the paged-cache attention operators (sym_amd.attention).

A serving step has four calls: the tables that say where the step's tokens go
(`block_tables`), the norm and rotation of its queries and keys
(`norm_rotate`, in training with `norm_rotate_backward`; in serving
`norm_rotate_append`, which puts keys and values into the cache), and the
attention of the step's tokens, one per request, a chunk or a drafted tree,
over the cache (`tree_attention`). A case is one of these calls.

`run` computes them in plain 32-bit torch operations, or through the package
where `own` is set. Request lengths are part of a case (they follow from its
values); the seed makes the tensors, the page order and the trees.
"""
import math
import random
import zlib

import torch

own = False

EPS = 1e-6
WORD = 64  # rows of a tree that one mask word holds
_contexts = {}


def _device():
    return torch.device("cuda", 0)


def _attention():
    """The package and one retained context, as a serving program keeps them."""
    if not _contexts:
        from sym_amd import attention, pyreloc
        _contexts["attention"], _contexts["context"] = attention, pyreloc.Context(0)
    return _contexts["attention"], _contexts["context"]


def listed():
    return [
        # one decoding step of a few requests: the tables' latency
        dict(name="tables 8x1", op="tables", requests=8, longest=4096, fresh=1, tree=False, page=16),
        # a speculative step: every request drafts a tree of up to 24 tokens
        dict(name="tables tree 64x24", op="tables", requests=64, longest=4096, fresh=24, tree=True, page=16),
        # admission of many prompts at once
        dict(name="tables prompts 1000x1024", op="tables", requests=1000, longest=0, fresh=1024, tree=False, page=64),
        # training, one micro-batch of eight sequences, queries and keys as views of the fused projection
        dict(name="rotate 8x4096", op="rotate", tokens=32768, heads=32, kv_heads=8, dim=128, rotary=128, pairs=False,
             dtype="bfloat16", back=False),
        dict(name="rotate back 8x4096", op="rotate", tokens=32768, heads=32, kv_heads=8, dim=128, rotary=128, pairs=False,
             dtype="bfloat16", back=True),
        # an odd head size, of which three quarters turn, in neighbouring pairs, over an odd number of tokens
        dict(name="rotate back odd 4099", op="rotate", tokens=4099, heads=12, kv_heads=4, dim=80, rotary=60, pairs=True,
             dtype="float16", back=True),
        # the serving form: 64 requests, one token each, and a chunk of a prompt into a head-major cache
        dict(name="append 64", op="append", tokens=64, heads=32, kv_heads=8, dim=128, rotary=128, pairs=False,
             dtype="bfloat16", page=16, order="slots"),
        dict(name="append 8192 head-major", op="append", tokens=8192, heads=32, kv_heads=32, dim=128, rotary=128, pairs=False,
             dtype="float16", page=64, order="heads"),
        # one request decodes alone: latency
        dict(name="attend 1x1 over 1024", op="attend", requests=1, longest=1024, fresh=1, tree=False, heads=32, kv_heads=8,
             dim=128, dtype="bfloat16", cache="bfloat16", page=16, order="slots"),
        # a full batch decodes over the int8 head-major cache that the package's cache plan lays out, one page a request
        dict(name="attend 64x1 int8", op="attend", requests=64, longest=4096, fresh=1, tree=False, heads=32, kv_heads=32,
             dim=128, dtype="float16", cache="int8", page=4096, order="heads"),
        # trees of 64 drafted tokens over long contexts: 256 query rows a key head
        dict(name="attend tree 8x64 over 8192", op="attend", requests=8, longest=8192, fresh=64, tree=True, heads=32,
             kv_heads=8, dim=128, dtype="bfloat16", cache="bfloat16", page=16, order="slots"),
        # one request, a small tree, a very long context: the work has to be split over it
        dict(name="attend tree 1x13 over 131072", op="attend", requests=1, longest=131072, fresh=13, tree=True, heads=32,
             kv_heads=8, dim=128, dtype="bfloat16", cache="bfloat16", page=256, order="slots"),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tables", "rotate", "append", "attend", "attend"])
    if op == "tables":
        tree = rng.random() < 0.5
        return dict(op=op, requests=_spread(rng, 1, 256 if tree else 1000), longest=rng.randint(0, 8192),
                    fresh=_spread(rng, 1, WORD if tree else 1024), tree=tree, page=rng.choice([1, 8, 16, 24, 64, 256]))
    kv_heads = rng.choice([1, 2, 4, 8, 32])
    dim = rng.choice([64, 80, 128, 128, 256] if op == "attend" else [64, 80, 96, 128, 128, 256])
    dtype = rng.choice(["bfloat16", "float16"])
    if op == "attend":
        heads = kv_heads * (1 if kv_heads == 32 else rng.choice([1, 3, 4, 8]))
        cache = rng.choice([dtype, dtype, "int8"])
        requests = _spread(rng, 1, 64)
        tree = rng.random() < 0.6
        fresh = _spread(rng, 1, WORD)
        # no more tokens than the largest listed cases hold, nor more scores in the plain form
        most = min(131072, 2 ** 31 // (requests * kv_heads * dim * 2 * (1 if cache == "int8" else 2)),
                   2 ** 30 // (requests * heads * fresh))
        return dict(op=op, requests=requests, longest=_spread(rng, 1, max(2, most)), fresh=fresh, tree=tree, heads=heads,
                    kv_heads=kv_heads, dim=dim, dtype=dtype, cache=cache, page=rng.choice([8, 16, 24, 64, 256]),
                    order=rng.choice(["slots", "heads"]))
    heads = kv_heads * rng.choice([1, 3, 4]) if kv_heads < 32 else 32
    tokens = _spread(rng, 1, min(65536, 32768 * 40 * 128 // ((heads + kv_heads) * dim)))
    case = dict(op=op, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                rotary=rng.choice([dim, dim, dim // 2, dim * 3 // 4]) // 2 * 2, pairs=rng.random() < 0.3, dtype=dtype)
    if op == "rotate":
        return dict(case, back=rng.random() < 0.5)
    return dict(case, tokens=min(tokens, 16384), page=rng.choice([8, 16, 24, 64, 256]), order=rng.choice(["slots", "heads"]))


def _lengths(case):
    """(cached, fresh) of every request: ragged where there are several, the longest as the case says."""
    key = repr(sorted((k, v) for k, v in case.items() if k != "name"))
    rng = random.Random(zlib.crc32(key.encode()))
    n, longest, fresh = case["requests"], case["longest"], case["fresh"]
    cached = [rng.randint(longest // 2, longest) for _ in range(n)]
    new = [rng.randint((fresh + 1) // 2, fresh) for _ in range(n)]
    cached[rng.randrange(n)], new[rng.randrange(n)] = longest, fresh
    return cached, new


def _pages(n, page):
    return -(-n // page)


def _tree(rng, n):
    """Parents of a drafted tree: each token follows one of the last few before it, or the context."""
    return [rng.randint(max(-1, j - 6), j - 1) for j in range(n)]


def _words(parents):
    """The ancestors of each token, itself among them, as one mask word."""
    rows = []
    for j, p in enumerate(parents):
        rows.append((1 << j) | (rows[p] if p >= 0 else 0))
    return [r - (1 << WORD) if r >> (WORD - 1) else r for r in rows]


def _order(case, gen, pages, width):
    """A cache of `pages` pages, [pages, page, kv_heads, width], slot-major or (viewed) head-major in memory."""
    page, heads = case["page"], case["kv_heads"]
    shape = (pages, page, heads, width) if case["order"] == "slots" else (pages, heads, page, width)
    if case.get("cache") == "int8":
        t = torch.randint(-100, 101, shape, generator=gen, device=_device(), dtype=torch.int8)
    else:
        t = torch.randn(shape, generator=gen, device=_device(), dtype=getattr(torch, case["dtype"]))
    return t if case["order"] == "slots" else t.transpose(1, 2)


def _page_table(gen, lengths, page, columns):
    """A table of pages in no order, -1 past each request's own, and how many pages the pool has."""
    need = [_pages(n, page) for n in lengths]
    pool = sum(need) + 3
    ids = torch.randperm(pool, generator=gen, device=_device(), dtype=torch.int64).to(torch.int32)
    counts = torch.tensor(need, device=_device())
    at = torch.arange(columns, device=_device())[None, :]
    first = (counts.cumsum(0) - counts)[:, None]
    table = torch.where(at < counts[:, None], ids[(first + at).clamp(max=pool - 1)], -1)
    return table.to(torch.int32).contiguous(), ids[sum(need):].contiguous(), pool


def _angles(positions, rotary):
    """cos and sin of a position table of the usual frequencies."""
    inv = 10000.0 ** (-torch.arange(0, rotary, 2, device=_device(), dtype=torch.float64) / rotary)
    a = torch.arange(positions, device=_device(), dtype=torch.float64)[:, None] * inv[None, :]
    return a.cos().float(), a.sin().float()


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=_device())


def prepare(case, seed):
    gen = torch.Generator(device=_device()).manual_seed(seed)
    rng = random.Random(seed)
    s = {"case": case}
    if case["op"] in ("tables", "attend"):
        cached, fresh = _lengths(case)
        s.update(rows=sum(fresh), cached=_ints(cached), fresh=_ints(fresh))
        trees = [_tree(rng, n) for n in fresh] if case["tree"] else None
    if case["op"] == "tables":
        columns = _pages(case["longest"] + case["fresh"], case["page"])
        s["table"], free, pool = _page_table(gen, cached, case["page"], columns)
        more = sum(_pages(c + f, case["page"]) for c, f in zip(cached, fresh))
        s["free"] = (torch.randperm(more + 2, generator=gen, device=_device()) + pool).to(torch.int32)
        s["parents"] = _ints([p for t in trees for p in t]) if trees else None
        return s
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    dtype = getattr(torch, case["dtype"])
    if case["op"] == "attend":
        lengths = [c + f for c, f in zip(cached, fresh)]
        columns = _pages(max(lengths), case["page"])
        s["table"], _, pool = _page_table(gen, lengths, case["page"], columns)
        s["starts"] = torch.cat([_ints([0]), s["fresh"].cumsum(0).to(torch.int32)])
        s["q"] = torch.randn((s["rows"], heads, dim), generator=gen, device=_device(), dtype=dtype)
        s["cache_k"], s["cache_v"] = _order(case, gen, pool, dim), _order(case, gen, pool, dim)
        s["mask"] = torch.tensor([w for t in trees for w in _words(t)], device=_device())[:, None] if trees else None
        s["scale"] = dim ** -0.5
        s["k_scale"] = s["v_scale"] = None
        if case["cache"] == "int8":
            s["k_scale"] = torch.rand(kv, generator=gen, device=_device()) * 0.02 + 0.01
            s["v_scale"] = torch.rand(kv, generator=gen, device=_device()) * 0.02 + 0.01
        s["most_rows"], s["most_tokens"] = max(fresh), max(lengths)
        return s
    n = case["tokens"]
    fused = torch.randn((n, (heads + 2 * kv) * dim), generator=gen, device=_device(), dtype=dtype)
    s["q"] = fused[:, :heads * dim].unflatten(1, (heads, dim))
    s["k"] = fused[:, heads * dim:(heads + kv) * dim].unflatten(1, (kv, dim))
    s["v"] = fused[:, (heads + kv) * dim:].unflatten(1, (kv, dim))
    length = min(n, 4096)
    s["positions"] = (torch.arange(n, device=_device()) % length).to(torch.int32)
    s["cos"], s["sin"] = _angles(length, case["rotary"])
    s["qw"] = (1 + 0.2 * torch.randn(dim, generator=gen, device=_device())).to(dtype)
    s["kw"] = (1 + 0.2 * torch.randn(dim, generator=gen, device=_device())).to(dtype)
    if case["op"] == "append":
        pages = _pages(n, case["page"]) + 2
        s["slots"] = torch.randperm(pages * case["page"], generator=gen, device=_device())[:n].contiguous()
        s["cache_k"], s["cache_v"] = _order(case, gen, pages, dim), _order(case, gen, pages, dim)
    elif case["back"]:
        s["dq"] = torch.randn((n, heads, dim), generator=gen, device=_device(), dtype=dtype)
        s["dk"] = torch.randn((n, kv, dim), generator=gen, device=_device(), dtype=dtype)
    return s


# ------------------------------------------------------------- plain forms

def _closure(reach):
    """Reachability in twice as many steps."""
    return (reach @ reach).clamp(max=1.0)


def _plain_tables(s):
    page, table, free = s["case"]["page"], s["table"], s["free"]
    cached, fresh, n = s["cached"].long(), s["fresh"].long(), s["rows"]
    requests, columns = table.shape
    starts = torch.cat([fresh.new_zeros(1), fresh.cumsum(0)])
    have = ((cached + page - 1) // page).clamp(max=columns)
    need = ((cached + fresh + page - 1) // page).clamp(max=columns) - have
    base = need.cumsum(0) - need
    row = torch.arange(n, device=table.device)
    req = torch.searchsorted(starts, row, right=True) - 1
    j = row - starts[req]
    x = cached[req] + j
    g = x // page
    old = table[req, g.clamp(max=columns - 1)].long()
    take = base[req] + g - have[req]
    new = torch.where(take < free.numel(), free[take.clamp(0, free.numel() - 1)].long(), -1)
    ids = torch.where(g < have[req], old, torch.where(g < columns, new, -1))
    slots = torch.where(ids >= 0, ids * page + x % page, -1)
    at = torch.arange(columns, device=table.device)[None, :]
    fill = base[:, None] + at - have[:, None]
    mine = (at >= have[:, None]) & (at < (have + need)[:, None])
    put = torch.where(fill < free.numel(), free[fill.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where(mine, put, table))
    out = [starts.to(torch.int32), slots, x.to(torch.int32), need.sum().to(torch.int32).reshape(1), table]
    if s["parents"] is None:
        return out
    # ancestors: the closure of "is a parent of", one matrix a request, 2^6 steps deep
    p = s["parents"].long()
    up = torch.zeros((requests, WORD, WORD), device=table.device)
    up[req, j, torch.where(p >= 0, p, j)] = 1.0
    up = (up + torch.eye(WORD, device=table.device)).clamp(max=1.0)
    reach = _closure(_closure(_closure(_closure(_closure(_closure(up))))))[req, j] > 0
    out[2] = (cached[req] + reach.sum(1) - 1).to(torch.int32)
    words = torch.where(reach, torch.ones((), dtype=torch.int64, device=table.device) << torch.arange(WORD, device=table.device), 0)
    return out + [words.sum(1)[:, None]]


def _turn(y, cos, sin, rotary, pairs, sign):
    """The rotation of the first `rotary` elements (sign -1: its transpose)."""
    r, rest = y[..., :rotary], y[..., rotary:]
    a, b = (r[..., 0::2], r[..., 1::2]) if pairs else (r[..., :rotary // 2], r[..., rotary // 2:])
    u, v = a * cos - sign * b * sin, b * cos + sign * a * sin
    r = torch.stack([u, v], -1).flatten(-2) if pairs else torch.cat([u, v], -1)
    return torch.cat([r, rest], -1)


def _plain_rotate(x, w, s, wide):
    c = s["case"]
    cos, sin = s["cos"].to(wide)[s["positions"].long()][:, None], s["sin"].to(wide)[s["positions"].long()][:, None]
    x = x.to(wide)
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    return _turn(n * w.to(wide), cos, sin, c["rotary"], c["pairs"], 1)


def _plain_back(dz, x, w, s, wide):
    c = s["case"]
    cos, sin = s["cos"].to(wide)[s["positions"].long()][:, None], s["sin"].to(wide)[s["positions"].long()][:, None]
    x, g = x.to(wide), _turn(dz.to(wide), cos, sin, c["rotary"], c["pairs"], -1)
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    n, u = x * r, g * w.to(wide)
    return r * (u - n * (u * n).mean(-1, keepdim=True)), (g * n).sum((0, 1))


def _plain_attend(s):
    c, q = s["case"], s["q"]
    heads, kv, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    group, rows, tokens = heads // kv, s["most_rows"], s["most_tokens"]
    cached, starts, table = s["cached"].long(), s["starts"].long(), s["table"].long()
    x = torch.arange(tokens, device=q.device)
    ids = table[:, x // page].clamp(min=0)
    k = s["cache_k"][ids, (x % page)[None, :]].float().transpose(1, 2)  # [B, kv, tokens, dim]
    v = s["cache_v"][ids, (x % page)[None, :]].float().transpose(1, 2)
    if s["k_scale"] is not None:
        k, v = k * s["k_scale"][:, None, None], v * s["v_scale"][:, None, None]
    j = torch.arange(rows, device=q.device)
    real = starts[:-1, None] + j[None, :] < starts[1:, None]
    at = (starts[:-1, None] + j[None, :]).clamp(max=q.shape[0] - 1)
    w = q.float()[at].unflatten(2, (kv, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, kv, group * rows, dim]
    d = x[None, None, :] - cached[:, None, None]  # the token's place among the fresh ones
    if s["mask"] is not None:
        bits = (s["mask"][at] >> d.clamp(0, WORD - 1)) & 1
        see = (d < 0) | ((d < WORD) & (bits > 0) & (d < (starts[1:] - starts[:-1])[:, None, None]))
    else:
        see = d <= j[None, :, None]
    see = (see & real[:, :, None])[:, None, None]
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
        if c["op"] == "tables":
            t = A.block_tables(ctx, s["cached"], s["fresh"], s["table"], s["free"], c["page"], s["rows"], parents=s["parents"])
            return [t.starts, t.slots, t.positions, t.taken, s["table"]] + ([t.mask] if s["parents"] is not None else [])
        if c["op"] == "attend":
            return A.tree_attention(ctx, s["q"], s["cache_k"], s["cache_v"], s["table"], s["cached"], s["starts"],
                                    mask=s["mask"], scale=s["scale"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        turn = (s["positions"], s["cos"], s["sin"], s["qw"], s["kw"], EPS)
        if c["op"] == "append":
            q = A.norm_rotate_append(ctx, s["q"], s["k"], s["v"], s["slots"], s["cache_k"], s["cache_v"], *turn, pairs=c["pairs"])
            return [q, s["cache_k"], s["cache_v"]]
        if c["back"]:
            return A.norm_rotate_backward(ctx, s["dq"], s["dk"], s["q"], s["k"], *turn, pairs=c["pairs"])
        return A.norm_rotate(ctx, s["q"], s["k"], *turn, pairs=c["pairs"])
    if c["op"] == "tables":
        return _plain_tables(s)
    if c["op"] == "attend":
        return _plain_attend(s)
    dtype, wide = s["q"].dtype, torch.float32
    if c["op"] == "rotate" and c["back"]:
        dq, dqw = _plain_back(s["dq"], s["q"], s["qw"], s, wide)
        dk, dkw = _plain_back(s["dk"], s["k"], s["kw"], s, wide)
        return [dq.to(dtype), dk.to(dtype), dqw, dkw]
    q, k = (_plain_rotate(s[x], s[x + "w"], s, wide).to(dtype) for x in "qk")
    if c["op"] == "rotate":
        return [q, k]
    page, off = s["slots"] // c["page"], s["slots"] % c["page"]
    s["cache_k"][page, off], s["cache_v"][page, off] = k, s["v"]
    return [q, s["cache_k"], s["cache_v"]]


def work(case):
    c = case
    if c["op"] == "tables":
        cached, fresh = _lengths(c)
        n = sum(fresh)
        new = sum(_pages(a + b, c["page"]) - _pages(a, c["page"]) for a, b in zip(cached, fresh))
        # lengths and starts; a slot, a position and (trees) a parent and a mask word a row; new pages from the list to the table
        return {"bytes": 12 * c["requests"] + n * (24 if c["tree"] else 12) + 8 * new, "flops": n}
    heads, kv, dim, width = c["heads"], c["kv_heads"], c["dim"], 2
    if c["op"] == "attend":
        cached, fresh = _lengths(c)
        cell = 1 if c["cache"] == "int8" else width
        tokens = sum(a + b for a, b in zip(cached, fresh))
        pages = sum(_pages(a + b, c["page"]) for a, b in zip(cached, fresh))
        scores = sum((a + b) * b for a, b in zip(cached, fresh))
        return {"bytes": 2 * tokens * kv * dim * cell + 2 * sum(fresh) * heads * dim * width + 4 * pages,
                "flops": 4 * scores * heads * dim}
    n = c["tokens"]
    turn = 4 * n + 8 * min(n, 4096) * (c["rotary"] // 2)
    moved = n * (heads + kv) * dim * width
    if c["op"] == "append":
        return {"bytes": 2 * moved + 2 * n * kv * dim * width + 8 * n + turn, "flops": 8 * n * (heads + kv) * dim}
    return {"bytes": (3 if c["back"] else 2) * moved + turn, "flops": (16 if c["back"] else 8) * n * (heads + kv) * dim}


# ---------------------------------------------- the definitions in 64 bits

def _exact_turn(y, s, sign):
    """Each pair of elements as a complex number, turned by its angle."""
    c = s["case"]
    r = c["rotary"]
    at = s["positions"].long()
    turn = torch.complex(s["cos"].double(), sign * s["sin"].double())[at][:, None, :]
    first = torch.arange(r // 2, device=y.device) * (2 if c["pairs"] else 1)
    second = first + (1 if c["pairs"] else r // 2)
    z = torch.complex(y[..., first], y[..., second]) * turn
    y = y.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_norm(x):
    x = x.double()
    return x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS)


def exact(case, seed):
    c = case
    if c["op"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    if c["op"] == "attend":
        q, outs = s["q"].double(), []
        starts, cached, table = s["starts"].tolist(), s["cached"].tolist(), s["table"].long()
        group = c["heads"] // c["kv_heads"]
        for b in range(c["requests"]):
            r0, r1 = starts[b], starts[b + 1]
            n = cached[b] + r1 - r0
            ids = table[b, :_pages(n, c["page"])]
            k = s["cache_k"][ids].flatten(0, 1)[:n].double()
            v = s["cache_v"][ids].flatten(0, 1)[:n].double()
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"].double()[:, None], v * s["v_scale"].double()[:, None]
            see = torch.ones((r1 - r0, n), dtype=torch.bool, device=q.device)
            for j in range(r1 - r0):
                if s["mask"] is None:
                    see[j, cached[b] + j + 1:] = False
                else:
                    word = int(s["mask"][r0 + j, 0]) & ((1 << WORD) - 1)
                    see[j, cached[b]:] = torch.tensor([bool(word >> i & 1) for i in range(r1 - r0)], device=q.device)
            heads = []
            for h in range(c["heads"]):
                a = (q[r0:r1, h] @ k[:, h // group].T * s["scale"]).masked_fill(~see, -math.inf)
                heads.append(torch.softmax(a, -1) @ v[:, h // group])
            outs.append(torch.stack(heads, 1))
        return torch.cat(outs)
    if c["op"] == "rotate" and c["back"]:
        outs = []
        for x, w, dz in (("q", "qw", "dq"), ("k", "kw", "dk")):
            leaf, weight = s[x].double().requires_grad_(), s[w].double().requires_grad_()
            outs.append(torch.autograd.grad(_exact_turn(_exact_norm(leaf) * weight, s, 1.0), (leaf, weight), s[dz].double()))
        return [outs[0][0], outs[1][0], outs[0][1], outs[1][1]]
    q, k = (_exact_turn(_exact_norm(s[x]) * s[x + "w"].double(), s, 1.0) for x in "qk")
    if c["op"] == "rotate":
        return [q, k]
    ck, cv = s["cache_k"].double(), s["cache_v"].double()
    page, off = s["slots"] // c["page"], s["slots"] % c["page"]
    ck[page, off], cv[page, off] = k, s["v"].double()
    return [q, ck, cv]
