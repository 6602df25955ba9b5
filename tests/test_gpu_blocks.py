"""Caches with a scale a block, and attention with a window over caches, on the GPU."""
import pytest

from tests import attention_cases as C
from tests import window_cases as W

torch = pytest.importorskip("torch")
from sym_amd import attention as A  # noqa: E402
from sym_amd import pyreloc as P  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32, I8 = torch.float16, torch.bfloat16, torch.float32, torch.int8


@pytest.fixture(scope="module")
def ctx():
    c = P.Context(0)
    yield c
    c.close()


def say(*what):
    print(*what, flush=True)


def on_gpu(s):
    """Every tensor on the GPU, views in their order of memory."""
    out = {}
    for k, v in s.items():
        if isinstance(v, torch.Tensor) and v.dim() == 4 and not v.is_contiguous():
            v = v.transpose(1, 2).to(DEV).transpose(1, 2)
        elif isinstance(v, torch.Tensor):
            v = v.to(DEV)
        out[k] = v
    return out


# ------------------------------------------------------------ appending

def append_case(seed, cached, fresh, kv, dim, dtype, page, block, order="slots", columns=None):
    s = W.view_case(seed, cached, fresh, kv, kv, dim, F16, I8, page, block, order, columns=columns)
    gen = torch.Generator().manual_seed(seed + 2)
    rows = sum(fresh)
    size = torch.exp(torch.randn((rows, kv, 1), generator=gen))
    s["k"] = (torch.randn((rows, kv, dim), generator=gen) * size).to(dtype)
    s["v"] = torch.randn((rows, kv, dim), generator=gen).to(dtype)
    return s


def check_append(ctx, s, what):
    say(what)
    want = W.block_append(*(s[n] for n in ("k", "v", "cache_k", "cache_v", "k_scale", "v_scale", "table", "cached", "starts")))
    d = on_gpu(s)
    A.block_append(ctx, *(d[n] for n in ("k", "v", "cache_k", "cache_v", "k_scale", "v_scale", "table", "cached", "starts")))
    for name, w in zip(("cache_k", "cache_v", "k_scale", "v_scale"), want):
        assert torch.equal(d[name].cpu(), w), (what, name)


@pytest.mark.parametrize("cached,fresh,kv,dim,dtype,page,block,order", [
    ([5], [1], 1, 64, BF16, 16, 16, "slots"),
    ([0, 16, 15, 47], [1, 1, 1, 1], 8, 128, BF16, 64, 16, "slots"),
    ([0, 3, 100], [70, 0, 33], 5, 80, F16, 48, 16, "heads"),
    ([31, 64, 7], [200, 1, 129], 4, 128, F32, 64, 64, "slots"),
    ([10], [300], 2, 256, BF16, 256, 128, "heads"),
    ([1, 2, 3], [40, 50, 60], 3, 24, F16, 32, 32, "slots"),
    ([9, 33], [77, 5], 2, 37, BF16, 32, 16, "slots"),
    ([3], [600], 1, 512, F32, 512, 512, "slots"),
])
def test_appending(ctx, cached, fresh, kv, dim, dtype, page, block, order):
    check_append(ctx, append_case(1, cached, fresh, kv, dim, dtype, page, block, order), "append %s" % [cached, fresh, dim])


@pytest.mark.parametrize("requests", [63, 64, 65, 130, 4500])
def test_appending_finds_the_requests(ctx, requests):
    fresh = [(i * 7) % 4 for i in range(requests)]
    cached = [(i * 13) % 40 for i in range(requests)]
    check_append(ctx, append_case(2, cached, fresh, 1, 8, BF16, 16, 16), "append, %d requests" % requests)


def test_what_is_appended_again_and_what_is_not_there(ctx):
    """Not finite, zero, tiny, out of the table, of no page; a scale of a block begun anew."""
    s = append_case(3, [20, 5, 0], [30, 40, 20], 2, 64, F32, 32, 16, columns=2)
    s["k"][3] = float("inf")
    s["k"][5, 0, 3] = float("nan")
    s["k"][40:60] = 0.0
    s["v"][70:] = 1e-44
    s["v"][10, 1, 5] = -float("inf")
    s["table"][1, 1] = -1
    s["table"][2, 0] = 10 ** 6
    s["k_scale"][int(s["table"][0, 1]), 0] = float("nan")  # of a block that the step begins
    check_append(ctx, s, "append, edges")


def test_appending_into_strided_scales_and_views(ctx):
    s = append_case(4, [12, 40], [9, 50], 4, 64, BF16, 64, 32)
    want = W.block_append(*(s[n] for n in ("k", "v", "cache_k", "cache_v", "k_scale", "v_scale", "table", "cached", "starts")))
    d = on_gpu(s)
    pages, blocks, kv = s["k_scale"].shape
    ks, vs = (torch.zeros((kv, pages, blocks + 1), device=DEV).permute(1, 2, 0)[:, :blocks] for _ in range(2))
    ks.copy_(d["k_scale"])
    vs.copy_(d["v_scale"])
    both = torch.stack([d["k"], d["v"]], 2)  # rows and heads of other strides
    wide = torch.zeros((2, 9), dtype=torch.int32, device=DEV)
    wide[:, :s["table"].shape[1]] = d["table"]
    A.block_append(ctx, both[:, :, 0], both[:, :, 1], d["cache_k"], d["cache_v"], ks, vs, wide[:, :s["table"].shape[1]],
                   d["cached"], d["starts"])
    for got, w in zip((d["cache_k"], d["cache_v"], ks, vs), want):
        assert torch.equal(got.cpu(), w)


# ------------------------------------------------------------ attention

def check_view(ctx, s, what, window=None, sinks=0, **more):
    say(what)
    want, lse, bound = W.view_attention(s["q"], s["cache_k"], s["cache_v"], s["table"], s["cached"], s["starts"], s["mask"],
                                        s["scale"], s["k_scale"], s["v_scale"], window, sinks, s["q"].dtype)
    d = on_gpu(s)
    got_lse = torch.full(s["q"].shape[:2], 7.0, device=DEV)
    got = A.tree_attention(ctx, d["q"], d["cache_k"], d["cache_v"], d["table"], d["cached"], d["starts"], mask=d["mask"],
                           scale=d["scale"], k_scale=d["k_scale"], v_scale=d["v_scale"], window=window, sinks=sinks,
                           lse=got_lse, **more)
    off = (got.cpu().double() - want).abs() - bound
    assert not torch.isnan(off).any() and float(off.max()) <= 0, (what, float(off.max()))
    far = (got_lse.cpu().double() - lse).abs()
    far = far[lse > -float("inf")]
    assert torch.equal(got_lse.cpu() == -float("inf"), lse == -float("inf")), what
    assert far.numel() == 0 or float(far.max()) < 2e-4, (what, float(far.max()))
    return got


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("cached,fresh,heads,kv,dim,page,block,order", [
    ([0], [1], 1, 1, 64, 16, 16, "slots"),
    ([1000], [1], 8, 2, 128, 64, 64, "slots"),
    ([5, 300, 31], [1, 1, 1], 4, 4, 80, 48, 16, "heads"),
    ([200, 77], [1, 2], 6, 2, 256, 32, 32, "slots"),
    ([500, 40], [40, 9], 8, 2, 128, 64, 32, "slots"),
    ([90], [130], 4, 1, 64, 128, 64, "heads"),
    ([3000], [3], 2, 1, 72, 64, 16, "slots"),
    ([300], [80], 8, 1, 128, 64, 16, "slots"),
])
def test_blocks(ctx, dtype, cached, fresh, heads, kv, dim, page, block, order):
    check_view(ctx, W.view_case(5, cached, fresh, heads, kv, dim, dtype, I8, page, block, order), "blocks %s" % [cached, fresh, dim])


@pytest.mark.parametrize("cached,fresh,heads,kv,dim,page,block,window,sinks", [
    ([700, 3, 129], [1, 1, 1], 16, 4, 128, 64, 32, None, 0),
    ([700, 0, 129], [2, 1, 1], 8, 8, 80, 64, 16, None, 0),
    ([5000, 31, 300], [1, 1, 1], 8, 4, 64, 48, 16, 1000, 3),
    ([300, 260, 900], [1, 2, 1], 12, 4, 128, 128, 64, 70, 40),
    ([90, 1000, 64], [9, 1, 0], 8, 8, 16, 64, 64, 33, 0),  # more rows of one request than fit at a time
    ([400, 200, 100], [1, 1, 1], 16, 16, 128, 64, None, 200, 1),  # a scale a head
])
def test_four_heads_at_a_time(ctx, cached, fresh, heads, kv, dim, page, block, window, sinks):
    """Decoding over many tokens whose heads lie side by side."""
    columns = (1 << 17) // (3 * page * kv) + 1
    for dtype in (F16, BF16):
        s = W.view_case(14, cached, fresh, heads, kv, dim, dtype, I8, page, block, columns=max(columns, 5100 // page + 1))
        got = check_view(ctx, s, "four heads %s" % [cached, fresh, dim, window], window, sinks)
        narrow = dict(s, table=s["table"][:, :max(-(-(c + f) // page) for c, f in zip(cached, fresh))].contiguous())
        other = check_view(ctx, narrow, "the same, one at a time", window, sinks)
        assert float((got.float() - other.float()).abs().max()) < 0.05


@pytest.mark.parametrize("kv,requests", [(8, 70), (4, 3)])
def test_small_tables(ctx, kv, requests):
    """Nothing is cut or joined; with many heads of many requests four at a time."""
    cached = [(i * 37) % 200 for i in range(requests)]
    fresh = [1 + (i == 2) for i in range(requests)]
    s = W.view_case(18, cached, fresh, kv, kv, 16, BF16, I8, 64, 16)
    check_view(ctx, s, "small tables", 90, 3)
    wide = on_gpu(s)
    rows = s["q"].shape[0]
    q = torch.cat([wide["q"], wide["q"], wide["q"]])  # rows of no request before and after
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=DEV)
    A.tree_attention(ctx, q, wide["cache_k"], wide["cache_v"], wide["table"], wide["cached"], wide["starts"] + rows,
                     scale=wide["scale"], k_scale=wide["k_scale"], v_scale=wide["v_scale"], window=90, sinks=3, out=out, lse=lse)
    assert not out[:rows].any() and not out[2 * rows:].any() and out[rows:2 * rows].any()
    assert (lse[:rows] == -float("inf")).all() and (lse[2 * rows:] == -float("inf")).all()
    none = torch.zeros((0, s["table"].shape[1]), dtype=torch.int32, device=DEV)
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = A.tree_attention(ctx, q, wide["cache_k"], wide["cache_v"], none, zero[:0], zero, k_scale=wide["k_scale"],
                           v_scale=wide["v_scale"])
    assert not got.any()


@pytest.mark.parametrize("cache", ["own", "int8", "blocks"])
@pytest.mark.parametrize("cached,fresh,heads,kv,dim,page,window,sinks", [
    ([0], [1], 2, 1, 64, 16, 1, 0),
    ([500], [1], 4, 1, 128, 16, 100, 4),
    ([500, 3, 129, 1000], [1, 1, 1, 1], 4, 2, 128, 64, 33, 1),
    ([2000], [1], 1, 1, 64, 32, 64, 70),
    ([400, 0], [50, 60], 8, 2, 128, 32, 40, 3),
    ([10, 700], [300, 5], 2, 1, 80, 64, 128, 17),
    ([90], [10], 2, 2, 256, 16, 4, 33),
    ([0, 40], [200, 100], 4, 1, 128, 64, 1, 2),
    ([600], [1], 4, 1, 128, 16, 10 ** 12, 10 ** 12),
    ([64], [1], 4, 1, 128, 16, 32, 1000),
])
def test_windows(ctx, cache, cached, fresh, heads, kv, dim, page, window, sinks):
    s = W.view_case(6, cached, fresh, heads, kv, dim, BF16, BF16 if cache == "own" else I8, page, 16 if cache == "blocks" else None)
    check_view(ctx, s, "window %s %s" % (cache, [cached, fresh, dim, window, sinks]), window, sinks)


@pytest.mark.parametrize("cache", ["own", "blocks"])
@pytest.mark.parametrize("words,fresh,window", [(1, [17, 64, 1], 64), (2, [100, 70, 3], 150)])
def test_windows_of_trees(ctx, cache, words, fresh, window):
    s = W.view_case(7, [300, 10, 900], fresh, 4, 2, 64, F16, F16 if cache == "own" else I8, 32, 32 if cache == "blocks" else None,
                    tree_words=words)
    check_view(ctx, s, "trees %s" % fresh, window, 5)


@pytest.mark.parametrize("page", [5, 24])
def test_windows_over_uneven_pages(ctx, page):
    for cache in (F16, I8):
        s = W.view_case(8, [100, 333], [1, 30], 4, 2, 64, F16, cache, page)
        check_view(ctx, s, "pages of %d" % page, 50, 9)


def test_what_no_row_sees_is_not_read_into_a_sum(ctx):
    """Tokens before the window, evicted pages, the rest of a block's tokens and scales
    of blocks behind the last token hold anything."""
    s = W.view_case(9, [600], [2], 4, 2, 64, BF16, BF16, 16)
    ids = s["table"][0].long()
    for p in range(1, 28):  # tokens 16 to 447; the window begins at 501
        s["cache_k"][ids[p]] = float("nan")
        s["cache_v"][ids[p]] = float("inf")
    s["cache_v"][ids[31], 4] = float("nan")  # token 500: just before both rows' windows
    s["cache_v"][ids[37], 10:] = float("nan")  # behind the last token
    gone = dict(s, table=s["table"].clone())
    gone["table"][0, 2:20] = -1
    for t, what in ((s, "not numbers"), (gone, "evicted")):
        got = check_view(ctx, dict(t, cache_k=t["cache_k"].nan_to_num(1.0), cache_v=t["cache_v"].nan_to_num(1.0, 1.0)),
                         what + ", as numbers", 100, 4)
        d = on_gpu(t)
        other = A.tree_attention(ctx, d["q"], d["cache_k"], d["cache_v"], d["table"], d["cached"], d["starts"],
                                 scale=d["scale"], window=100, sinks=4)
        assert torch.equal(got, other), what
    s = W.view_case(10, [40, 70], [1, 40], 4, 2, 64, F16, I8, 64, 16)
    d = on_gpu(s)
    args = [d["q"], d["cache_k"], d["cache_v"], d["table"], d["cached"], d["starts"]]
    see = dict(scale=d["scale"], window=20, sinks=1)
    want = A.tree_attention(ctx, *args, k_scale=d["k_scale"], v_scale=d["v_scale"], **see)
    for z in (d["k_scale"], d["v_scale"]):
        z[d["table"][0, 0].long(), 3] = float("nan")  # blocks of no token of the request
        z[d["table"][1, 1].long(), 3] = float("inf")
    assert torch.equal(want, A.tree_attention(ctx, *args, k_scale=d["k_scale"], v_scale=d["v_scale"], **see))


def test_a_value_that_is_not_finite_reaches_the_rows_that_see_it(ctx):
    """In a window that some rows' tiles share."""
    s = W.view_case(11, [200], [12], 2, 1, 64, BF16, BF16, 16)
    x = 200 + 3 - 40 + 1  # the first token of row 3's window of 40
    s["cache_v"][s["table"][0, x // 16].long(), x % 16, 0, 5] = float("inf")
    d = on_gpu(s)
    got = A.tree_attention(ctx, d["q"], d["cache_k"], d["cache_v"], d["table"], d["cached"], d["starts"], window=40).cpu()
    assert torch.isinf(got[:4, :, 5]).all() and torch.isfinite(got[4:]).all()
    assert torch.isfinite(got[:4, :, :5]).all() and torch.isfinite(got[:4, :, 6:]).all()


def test_large_and_small_scales_in_f16(ctx):
    """Weights are scaled by their values' scales before they are rounded to f16."""
    for size in (1e-7, 30.0, 3000.0):
        s = W.view_case(12, [300], [3], 4, 1, 64, F16, I8, 64, 16)
        s["v_scale"] = s["v_scale"] * (size / float(s["v_scale"].max()))
        if size > 100:  # results within f16
            s["cache_v"] = (s["cache_v"].float() / 64).to(I8)
            s["v_scale"] /= 4
        check_view(ctx, s, "scales of %g" % size, 200, 2)
    s = W.view_case(13, [300], [3], 4, 1, 64, F16, I8, 64, 16)
    s["v_scale"][:, 0] *= 1e4  # far apart, the small ones first and last
    s["k_scale"][:, 1] = 0.0
    s["v_scale"][:, 1] = 0.0
    s["cache_v"] = (s["cache_v"].float() / 16).to(I8)
    check_view(ctx, s, "scales far apart")


@pytest.mark.parametrize("scale", [0.05, -0.05, 0.0])
def test_scales_of_either_sign(ctx, scale):
    """Of the scores, and of an int8 cache's keys and values, a head's or a block's."""
    for block in (None, 16):
        for fresh in ([1, 1], [30, 7]):
            s = W.view_case(15, [200, 50], fresh, 4, 4, 64, BF16, I8, 32, block)
            s["scale"] = scale
            for z in (s["k_scale"], s["v_scale"]):
                z[..., 1] *= -1
                z[..., 2] = 0.0
            check_view(ctx, s, "scales %s %s" % (scale, block), 64, 2)


def test_windows_beyond_any_number(ctx):
    s = W.view_case(16, [100], [1], 2, 1, 64, F16, F16, 16)
    check_view(ctx, s, "all", 10 ** 30, 10 ** 30)


def test_a_step_over_blocks(ctx):
    """Tables, norm and rotation, appending, attention: prompts, then single tokens, captured and replayed."""
    say("a step over blocks")
    gen = torch.Generator().manual_seed(4)
    heads, kv, dim, page, block, requests = 8, 2, 64, 32, 16, 3
    lengths = [40, 5, 70]
    pool = 16
    cache = [torch.zeros((pool, page, kv, dim), dtype=I8, device=DEV) for _ in range(2)]
    scale = [torch.zeros((pool, page // block, kv), device=DEV) for _ in range(2)]
    table = torch.full((requests, 4), -1, dtype=torch.int32, device=DEV)
    free = torch.arange(pool, dtype=torch.int32, device=DEV).flip(0).contiguous()
    at = torch.arange(256)[:, None] * 10000.0 ** (-torch.arange(dim // 2) / (dim // 2))
    cos, sin = at.cos().float().to(DEV), at.sin().float().to(DEV)
    weight = torch.ones(dim, dtype=BF16, device=DEV)
    host_k, host_v = [[] for _ in range(requests)], [[] for _ in range(requests)]

    def step(q, k, v, cached, fresh, rows):
        t = A.block_tables(ctx, cached, fresh, table, free, page, rows)
        q, k = A.norm_rotate(ctx, q, k, t.positions, cos, sin, weight, weight, 1e-6)
        A.block_append(ctx, k, v, cache[0], cache[1], scale[0], scale[1], table, cached, t.starts)
        return q, k, t, A.tree_attention(ctx, q, cache[0], cache[1], table, cached, t.starts, k_scale=scale[0],
                                         v_scale=scale[1], window=48, sinks=2)

    def check(q, k, v, t, out, cached):
        starts = t.starts.cpu()
        for b in range(requests):
            host_k[b].append(k[int(starts[b]):int(starts[b + 1])].cpu())
            host_v[b].append(v[int(starts[b]):int(starts[b + 1])].cpu())
        want, _, bound = W.view_attention(q.cpu(), cache[0].cpu(), cache[1].cpu(), table.cpu(), cached.cpu(), starts, None,
                                          dim ** -0.5, scale[0].cpu(), scale[1].cpu(), 48, 2, BF16)
        assert float(((out.cpu().double() - want).abs() - bound).max()) <= 0
        for b in range(requests):  # every token within half a step of its block's scale, or one and a half if rounded anew
            n = sum(len(x) for x in host_k[b])
            ids = table[b, :-(-n // page)].long().cpu()
            for c, z, host in zip(cache, scale, (host_k, host_v)):
                held = W.values(c.cpu()[ids], z.cpu()[ids]).flatten(0, 1)[:n]
                step_size = z.cpu()[ids].repeat_interleave(block, 1).flatten(0, 1)[:n].double()
                assert ((held - torch.cat(host[b]).double()).abs() <= 4 * step_size[..., None]).all()

    def new(rows):
        return [torch.randn((rows, h, dim), generator=gen).to(BF16).to(DEV) for h in (heads, kv, kv)]
    zeros = torch.zeros(requests, dtype=torch.int32, device=DEV)
    fresh = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    q, k, v = new(sum(lengths))
    qt, kt, t, out = step(q, k, v, zeros, fresh, sum(lengths))
    check(qt, kt, v, t, out, zeros)
    free = free[int(t.taken):].contiguous()
    cached, one = fresh.clone(), torch.ones(requests, dtype=torch.int32, device=DEV)
    q, k, v = new(requests)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    saved = [x.clone() for x in (*cache, *scale, table)]
    with torch.cuda.stream(side):
        step(q, k, v, cached, one, requests)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip((*cache, *scale, table), saved):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qt, kt, t, out = step(q, k, v, cached, one, requests)
    for _ in range(3):
        for x, y in zip((q, k, v), new(requests)):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert int(t.taken) == 0
        check(qt, kt, v, t, out, cached)
        cached += 1


# ------------------------------------------------------------ refusals

def test_refusals(ctx):
    say("refusals")
    s = on_gpu(append_case(1, [20], [2], 2, 64, F16, 32, 16))

    def go(**more):
        d = dict(s, **more)
        return A.block_append(ctx, *(d[n] for n in ("k", "v", "cache_k", "cache_v", "k_scale", "v_scale", "table", "cached", "starts")))
    go()
    for bad in (dict(k=s["k"].to(I8)), dict(k=s["k"].cpu()), dict(v=s["v"].float()), dict(v=s["v"][:1]), dict(k=s["k"][:, :1]),
                dict(cache_k=s["cache_k"].half(), cache_v=s["cache_v"].half()), dict(cache_v=s["cache_v"][:1]),
                dict(k_scale=s["k_scale"][:1]), dict(k_scale=s["k_scale"].double()), dict(k_scale=s["k_scale"][:, :, 0]),
                dict(v_scale=s["v_scale"].transpose(0, 1).contiguous().transpose(0, 1)),
                dict(table=s["table"].long()), dict(cached=s["cached"].long()), dict(starts=s["starts"][:1])):
        with pytest.raises(ValueError):
            go(**bad)
    small = torch.ones((s["cache_k"].shape[0], 4, 2), device=DEV)  # blocks of 8
    with pytest.raises(P.TransferError, match="unsupported_layout"):
        go(k_scale=small, v_scale=small)
    one = torch.ones((1, 1, 1), device=DEV).expand(s["k_scale"].shape)
    with pytest.raises(P.TransferError, match="invalid_argument"):
        go(k_scale=one, v_scale=one)
    t = on_gpu(W.view_case(1, [20], [2], 4, 2, 64, F16, I8, 32, 16, tree_words=1))

    def attend(**more):
        d = dict(dict(t, window=None, sinks=0), **more)
        return A.tree_attention(ctx, d["q"], d["cache_k"], d["cache_v"], d["table"], d["cached"], d["starts"], mask=d["mask"],
                                k_scale=d["k_scale"], v_scale=d["v_scale"], window=d["window"], sinks=d["sinks"])
    attend()
    attend(window=64, sinks=3)
    for bad in (dict(window=-1), dict(sinks=3), dict(window=64, sinks=-1), dict(v_scale=None), dict(v_scale=t["v_scale"][:, :, :1]),
                dict(cache_k=t["cache_k"].half(), cache_v=t["cache_v"].half()), dict(window=0, sinks=2)):
        with pytest.raises(ValueError):
            attend(**bad)
    with pytest.raises(P.TransferError, match="unsupported_layout"):
        attend(window=63)
    with pytest.raises(P.TransferError, match="unsupported_layout"):
        attend(k_scale=small, v_scale=small)
    q = t["q"].clone().requires_grad_()
    out = A.tree_attention(ctx, q, t["cache_k"], t["cache_v"], t["table"], t["cached"], t["starts"], k_scale=t["k_scale"],
                           v_scale=t["v_scale"], window=9)
    with pytest.raises(RuntimeError, match="no gradient"):
        out.float().sum().backward()
