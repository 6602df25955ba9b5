"""The paged-cache operators on the MI355X against their definitions in 64
bits (tests/attention_cases.py), at the sizes, masks, strides and lengths
where they can go wrong. Bounds come from the number and size of the roundings
(see there), not from runs."""
import sys

import numpy as np
import pytest

from tests import attention_cases as C

torch = pytest.importorskip("torch")
from sym_amd import attention as A  # noqa: E402
from sym_amd import pyreloc as P  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-6
F16, BF16, F32, I8 = torch.float16, torch.bfloat16, torch.float32, torch.int8


def say(*a):
    print("[gpu-case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ctx():
    assert torch.cuda.is_available(), "a GPU test needs the MI355X"
    c = P.Context(0)
    yield c
    c.close()


def within(got, want, bound, what):
    got, want = got.double().cpu(), want.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    ok = torch.nan_to_num((got - want).abs()) <= torch.nan_to_num(bound.cpu())
    worst = ((got - want).abs() / bound.clamp(min=1e-300).cpu()).nan_to_num(0).max()
    assert bool(ok.all()), (what, "error over bound", float(worst), int((~ok).sum()), "of", ok.numel())


# ------------------------------------------------------------ block tables

def run_tables(ctx, cached, fresh, page, columns, free, rows=None, parents=None, words=1, out=False):
    total = sum(max(f, 0) for f in fresh)
    rows = total if rows is None else rows
    rng = np.random.default_rng(1)
    table = np.full((len(cached), columns), -1, np.int32)
    for b, c in enumerate(cached):
        n = min(columns, -(-max(c, 0) // page))
        table[b, :n] = rng.integers(0, 1 << 20, n)
    want = C.tables(cached, fresh, table, free, page, rows, parents, words if parents is not None else 0)
    t = torch.from_numpy(table).to(DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    given = None
    if out:
        given = A.Tables(torch.full((len(cached) + 1,), -7, **i32), torch.full((rows,), -7, dtype=torch.int64, device=DEV),
                         torch.full((rows,), -7, **i32), torch.full((1,), -7, **i32),
                         torch.full((rows, words), -7, dtype=torch.int64, device=DEV) if parents is not None else None)
    p = None if parents is None else torch.tensor(parents + [0] * (rows - len(parents)), **i32)
    got = A.block_tables(ctx, torch.tensor(cached, **i32), torch.tensor(fresh, **i32), t, torch.tensor(free, **i32), page,
                         rows, parents=p, words=words, out=given)
    torch.cuda.synchronize()
    assert got.starts.tolist() == want[0]
    assert got.slots.tolist() == want[1]
    assert got.positions.tolist() == want[2]
    assert got.taken.tolist() == [want[3]]
    if rows >= total:
        assert t.tolist() == [list(map(int, r)) for r in want[4]]
    if parents is None:
        assert got.mask is None
    else:
        assert got.mask.tolist() == want[5]


@pytest.mark.parametrize("requests,page,most,fresh", [
    (1, 1, 5, 1), (1, 16, 0, 1), (1, 16, 16, 1), (1, 16, 15, 3), (7, 16, 100, 1), (64, 24, 300, 40), (255, 8, 50, 9),
    (256, 8, 50, 9), (257, 8, 50, 9), (1000, 64, 4096, 30), (2500, 3, 20, 4), (3, 256, 70000, 2000)])
def test_block_tables(ctx, requests, page, most, fresh):
    say("tables", requests, page, most, fresh)
    rng = np.random.default_rng(requests * 7 + page)
    cached = rng.integers(0, most + 1, requests).tolist()
    new = rng.integers(0, fresh + 1, requests).tolist()
    columns = -(-(most + fresh) // page)
    wants = sum(-(-(c + f) // page) - -(-c // page) for c, f in zip(cached, new))
    free = rng.permutation(wants + 5).tolist()
    run_tables(ctx, cached, new, page, columns, free)


@pytest.mark.parametrize("fresh,words", [(1, 1), (24, 1), (64, 1), (65, 2), (150, 3), (150, 2), (40, 3)])
def test_block_tables_of_trees(ctx, fresh, words):
    say("trees", fresh, words)
    import random
    rng = random.Random(fresh)
    new = [rng.randint(0, fresh) for _ in range(9)] + [fresh]
    cached = [rng.randint(0, 90) for _ in new]
    parents = [p for n in new for p in C.tree(rng, n)]
    run_tables(ctx, cached, new, 16, 40, list(range(100, 300)), parents=parents, words=words, out=fresh == 24)


def test_block_tables_of_a_chain_and_of_bad_parents(ctx):
    say("chain, bad parents")
    run_tables(ctx, [5], [130], 16, 20, list(range(50)), parents=[j - 1 for j in range(130)], words=3)
    # a parent that is not an earlier token counts as the context
    run_tables(ctx, [5, 0], [6, 4], 16, 20, list(range(50)), parents=[-1, 0, 2, 99, -5, 1, 0, 0, 3, 1], words=1)


def test_block_tables_edges(ctx):
    say("edges")
    run_tables(ctx, [], [], 16, 4, [3])
    run_tables(ctx, [4, 0], [0, 0], 16, 4, [3])                                  # nothing new
    run_tables(ctx, [4, -3, 7], [2, 5, -2], 16, 4, [3, 1, 2])                    # negative lengths are none
    run_tables(ctx, [10, 10], [40, 40], 16, 8, [9, 8])                           # the list runs out
    run_tables(ctx, [10, 10], [40, 40], 16, 8, [])                               # and an empty one
    run_tables(ctx, [60, 3], [10, 4], 16, 4, [7, 8])                             # past the table's columns
    run_tables(ctx, [3, 4], [2, 3], 16, 4, [7, 8], rows=11)                      # rows of no request
    run_tables(ctx, [3, 4], [2, 3], 16, 4, [7, 8], rows=12, parents=[-1, 0, -1, 0, 0], words=2)
    run_tables(ctx, [3, 40], [20, 30], 16, 8, [7, 8, 9, 10], rows=30)            # more rows than the step may have
    run_tables(ctx, [3, 4], [2, 3], 16, 4, [7, 8], rows=0)


# --------------------------------------------------------- norm and rotation

def heads_of(gen, rows, heads, dim, dtype, layout):
    """[rows, heads, dim] on the GPU: dense, a view of a fused row, or head-major."""
    if layout == "fused":
        t = torch.randn((rows, (heads + 3) * dim + 5), generator=gen).to(dtype).to(DEV)
        return t[:, 2 * dim + 5:(heads + 2) * dim + 5].unflatten(1, (heads, dim))
    if layout == "heads":
        return torch.randn((heads, rows, dim), generator=gen).to(dtype).to(DEV).transpose(0, 1)
    return torch.randn((rows, heads, dim), generator=gen).to(dtype).to(DEV)


def rotation(seed, rows, heads, kv, dim, rotary, dtype, layout="dense", weight=F32, angles=97):
    gen = torch.Generator().manual_seed(seed)
    s = dict(q=heads_of(gen, rows, heads, dim, dtype, layout), k=heads_of(gen, rows, kv, dim, dtype, layout))
    s["positions"] = torch.randint(0, angles, (rows,), generator=gen, dtype=torch.int32).to(DEV)
    a = torch.rand((angles, rotary // 2), generator=gen, dtype=torch.float64) * 6.28
    s["cos"], s["sin"] = a.cos().float().to(DEV), a.sin().float().to(DEV)
    s["q_weight"] = s["k_weight"] = None
    if weight is not None:
        s["q_weight"], s["k_weight"] = ((1 + 0.3 * torch.randn(dim, generator=gen)).to(weight).to(DEV) for _ in range(2))
    return s


def turned(s):
    """cos and sin of every row in 64 bits, on the CPU."""
    p = s["positions"].cpu().long()
    return s["cos"].cpu().double()[p], s["sin"].cpu().double()[p]


def check_rotated(got, x, w, s, rotary, pairs, what):
    w = None if w is None else w.cpu()
    z, bound = C.norm_rotate(x.cpu(), w, *turned(s), rotary, pairs, EPS)
    u = C.ROUND[x.dtype]
    within(got, z, bound * (1 + u) + u * z.abs() + (2.0 ** -25 if x.dtype == F16 else 0), what)


ROTATIONS = [
    # rows, heads, kv, dim, rotary, pairs
    (1, 1, 1, 8, 8, False), (3, 2, 1, 64, 64, False), (33, 32, 8, 128, 128, False), (17, 5, 5, 128, 64, False),
    (29, 12, 4, 80, 60, False), (29, 12, 4, 80, 60, True), (9, 3, 1, 96, 72, False), (40, 9, 3, 256, 256, False),
    (13, 4, 2, 256, 192, True), (7, 2, 2, 512, 512, False), (11, 3, 3, 72, 20, True), (19, 7, 2, 50, 26, False),
    (5, 2, 1, 7, 6, False), (5, 2, 1, 7, 2, True), (21, 33, 3, 64, 0, False), (300, 8, 1, 320, 16, False),
    (2000, 4, 4, 64, 32, True)]


@pytest.mark.parametrize("rows,heads,kv,dim,rotary,pairs", ROTATIONS)
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_norm_rotate(ctx, rows, heads, kv, dim, rotary, pairs, dtype):
    for layout, weight in (("dense", F32), ("fused", dtype), ("heads", None)):
        say("rotate", rows, heads, kv, dim, rotary, pairs, dtype, layout, weight)
        s = rotation(rows + dim, rows, heads, kv, dim, rotary, dtype, layout, weight)
        q, k = A.norm_rotate(ctx, s["q"], s["k"], s["positions"], s["cos"], s["sin"], s["q_weight"], s["k_weight"], EPS,
                             pairs=pairs)
        torch.cuda.synchronize()
        check_rotated(q, s["q"], s["q_weight"], s, rotary, pairs, (layout, "q"))
        check_rotated(k, s["k"], s["k_weight"], s, rotary, pairs, (layout, "k"))


def test_norm_rotate_in_place_and_bad_positions(ctx):
    say("in place, bad positions")
    s = rotation(3, 20, 4, 2, 128, 64, BF16)
    args = (s["positions"], s["cos"], s["sin"], s["q_weight"], s["k_weight"], EPS)
    q, k = A.norm_rotate(ctx, s["q"], s["k"], *args)
    q2, k2 = s["q"].clone(), s["k"].clone()
    assert A.norm_rotate(ctx, q2, k2, *args, out=(q2, k2))[0] is q2
    torch.cuda.synchronize()
    assert torch.equal(q, q2) and torch.equal(k, k2)
    s["positions"][5], s["positions"][9] = -1, 97
    q3, _ = A.norm_rotate(ctx, s["q"], s["k"], *args)
    torch.cuda.synchronize()
    bad = torch.zeros(20, dtype=torch.bool, device=DEV)
    bad[5] = bad[9] = True
    assert torch.isnan(q3[bad][..., :64]).all() and torch.equal(q3[bad][..., 64:], q[bad][..., 64:])
    assert torch.equal(q3[~bad], q[~bad])


def test_norm_rotate_of_nothing(ctx):
    say("no rows, no heads")
    s = rotation(4, 0, 4, 2, 64, 64, F16)
    args = (s["positions"], s["cos"], s["sin"], s["q_weight"], s["k_weight"], EPS)
    assert A.norm_rotate(ctx, s["q"], s["k"], *args)[0].shape == (0, 4, 64)
    gq, gk, gqw, gkw = A.norm_rotate_backward(ctx, s["q"], s["k"], s["q"], s["k"], *args)
    assert gq.shape == (0, 4, 64) and not gqw.any() and not gkw.any()
    s = rotation(4, 5, 4, 0, 64, 64, F16)
    gq, gk, gqw, gkw = A.norm_rotate_backward(ctx, s["q"], s["k"], s["q"], s["k"], s["positions"], s["cos"], s["sin"],
                                              s["q_weight"], s["k_weight"], EPS)
    torch.cuda.synchronize()
    assert gk.shape == (5, 0, 64) and not gkw.any() and gqw.any()


@pytest.mark.parametrize("rows,heads,kv,dim,rotary,pairs", ROTATIONS)
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_norm_rotate_backward(ctx, rows, heads, kv, dim, rotary, pairs, dtype):
    for layout, weight in (("dense", dtype), ("fused", F32), ("heads", None)):
        say("rotate back", rows, heads, kv, dim, rotary, pairs, dtype, layout, weight)
        s = rotation(rows + dim, rows, heads, kv, dim, rotary, dtype, layout, weight)
        gen = torch.Generator().manual_seed(rows)
        dq, dk = heads_of(gen, rows, heads, dim, dtype, layout), heads_of(gen, rows, kv, dim, dtype, layout)
        got = A.norm_rotate_backward(ctx, dq, dk, s["q"], s["k"], s["positions"], s["cos"], s["sin"], s["q_weight"],
                                     s["k_weight"], EPS, pairs=pairs)
        torch.cuda.synchronize()
        u = C.ROUND[dtype]
        for x, dz, g, gw in (("q", dq, got[0], got[2]), ("k", dk, got[1], got[3])):
            w = s[x + "_weight"]
            want, bound, want_w, size_w = C.norm_rotate_back(dz.cpu(), s[x].cpu(), None if w is None else w.cpu(), *turned(s),
                                                             rotary, pairs, EPS)
            within(g, want, bound * (1 + u) + u * want.abs() + (2.0 ** -25 if dtype == F16 else 0), (layout, x))
            if w is None:
                assert gw is None
            else:
                # a term has dim / 2 + 8 roundings, a block's sum fewer than 64 terms in a row
                # here, and the blocks' parts are added in sixteens
                within(gw, want_w, (dim / 2 + 8 + 64 + 128) * C.F32 * size_w, (layout, x, "weight"))


def test_norm_rotate_gradient_against_differences(ctx):
    """Central differences of the 32-bit forward pass along random directions:
    the step's truncation is h^2 / 6 of the third derivative along the unit-sized
    direction (the norm's is below 15 / |x|^3, |x| here about 8), the rounding
    2^-22 of the sum of the terms over h."""
    say("differences")
    s = rotation(8, 6, 3, 2, 64, 48, F32)
    args = (s["positions"], s["cos"], s["sin"])
    gen = torch.Generator().manual_seed(5)
    dq, dk = (torch.randn(s[x].shape, generator=gen).to(DEV) for x in "qk")
    gq, gk, gqw, gkw = A.norm_rotate_backward(ctx, dq, dk, s["q"], s["k"], *args, s["q_weight"], s["k_weight"], EPS)
    for what, grad in (("q", gq), ("k", gk), ("q_weight", gqw), ("k_weight", gkw)):
        d = torch.randn(s[what].shape, generator=gen).to(DEV)
        h = 2.0 ** -7
        total, size = 0.0, 0.0
        for sign in (1, -1):
            t = dict(s, **{what: s[what] + sign * h * d})
            zq, zk = A.norm_rotate(ctx, t["q"], t["k"], *args, t["q_weight"], t["k_weight"], EPS)
            terms = [(zq.double() * dq.double()), (zk.double() * dk.double())]
            total += sign * float(sum(x.sum() for x in terms))
            size += float(sum(x.abs().sum() for x in terms))
        want = float((grad.double() * d.double()).sum())
        limit = h * h / 6 * 15 * float(d.norm()) ** 3 / 8 + 2.0 ** -22 * size / (2 * h)
        assert abs(total / (2 * h) - want) <= limit, (what, total / (2 * h), want, limit)


def test_norm_rotate_autograd(ctx):
    """Through torch's graph: broadcast inputs and weights shared by several calls add up."""
    say("autograd")
    s = rotation(9, 10, 4, 2, 64, 64, F32)
    args = (s["positions"], s["cos"], s["sin"])
    base = s["q"][:, :1].clone().requires_grad_()
    k = s["k"].clone().requires_grad_()
    w = s["q_weight"].clone().requires_grad_()
    zq, zk = A.norm_rotate(ctx, base.expand(10, 4, 64), k, *args, w, w, EPS)
    dq, dk = torch.randn_like(zq), torch.randn_like(zk)
    ((zq * dq).sum() + (zk * dk).sum()).backward()
    gq, gk, gqw, gkw = A.norm_rotate_backward(ctx, dq, dk, base.detach().expand(10, 4, 64), k.detach(), *args, w.detach(),
                                              w.detach(), EPS)
    torch.cuda.synchronize()
    assert torch.allclose(base.grad, gq.sum(1, keepdim=True), rtol=1e-5, atol=1e-5)
    assert torch.equal(k.grad, gk)
    assert torch.allclose(w.grad, gqw + gkw, rtol=1e-6, atol=1e-5)
    z = A.norm_rotate(ctx, base.detach().expand(10, 4, 64), k.detach(), *args, w.detach(), w.detach(), EPS)
    assert torch.equal(z[0], zq) and not z[0].requires_grad


@pytest.mark.parametrize("dim,page,order,dtype,cache", [
    (128, 16, "slots", BF16, BF16), (128, 16, "heads", F16, F16), (64, 24, "slots", F16, I8), (80, 7, "heads", BF16, I8),
    (256, 64, "heads", BF16, I8), (50, 5, "slots", F32, F32), (128, 64, "heads", F32, I8), (9, 3, "slots", F16, I8)])
def test_append(ctx, dim, page, order, dtype, cache):
    say("append", dim, page, order, dtype, cache)
    rows, heads, kv = 37, 6, 3
    rotary = dim // 2 // 2 * 2
    s = rotation(dim + page, rows, heads, kv, dim, rotary, dtype, "fused", dtype)
    gen = torch.Generator().manual_seed(dim)
    v = heads_of(gen, rows, kv, dim, dtype, "fused")
    pages = 60 // page + 2
    shape = (pages, page, kv, dim) if order == "slots" else (pages, kv, page, dim)
    before = [torch.randint(-100, 100, shape, generator=gen).to(cache) for _ in range(2)]
    now = [b.to(DEV) for b in before]
    if order == "heads":
        before, now = [b.transpose(1, 2) for b in before], [b.transpose(1, 2) for b in now]
    slots = torch.randperm(pages * page, generator=gen)[:rows]
    slots[3], slots[8], slots[30] = -1, pages * page, 1 << 40  # none of them a slot of the cache
    scales = [(torch.rand(kv, generator=gen) * 0.03 + 0.01) for _ in range(2)] if cache is I8 else [None, None]
    dev = [None if x is None else x.to(DEV) for x in scales]
    q = A.norm_rotate_append(ctx, s["q"], s["k"], v, slots.to(DEV), now[0], now[1], s["positions"], s["cos"], s["sin"],
                             s["q_weight"], s["k_weight"], EPS, k_scale=dev[0], v_scale=dev[1])
    torch.cuda.synchronize()
    check_rotated(q, s["q"], s["q_weight"], s, rotary, False, "q")
    z, bound = C.norm_rotate(s["k"].cpu(), s["k_weight"].cpu(), *turned(s), rotary, False, EPS)
    u = C.ROUND[dtype]
    live = [i for i in range(rows) if 0 <= int(slots[i]) < pages * page]
    at = slots[live]
    for kind, (got, old, exact, b) in enumerate(zip(now, before, (z, v.cpu().double()), (bound, torch.zeros_like(z)))):
        got, want = got.cpu(), old.clone()
        rowsof = got[at // page, at % page].double()
        if cache is I8:
            inv = (1.0 / scales[kind].double())[:, None]
            t = (exact[live] * inv).clamp(-128, 127)
            # off by the value's own error at most, and by the scale's and the product's rounding
            limit = 0.5 + (b[live] * inv) + 3 * C.F32 * t.abs()
            assert bool(((rowsof - t).abs() <= limit).all()), kind
        elif kind == 1:
            assert torch.equal(rowsof, exact[live])  # values as they are
        else:
            within(rowsof, exact[live], b[live] * (1 + u) + u * exact[live].abs() + 2.0 ** -25, "k")
        want[at // page, at % page] = got[at // page, at % page]
        assert torch.equal(got, want)  # and nothing else


def test_append_in_place_and_quantizes_as_the_plans_do(ctx):
    """Values whose products with 1 / scale fall on halves, out of range, on
    NaN and infinities, beside the package's quantize plan of the same rows."""
    say("append quantizes")
    from sym_amd import encoder as EN
    rows, kv, dim = 16, 2, 64
    gen = torch.Generator().manual_seed(1)
    v = (torch.randint(-300, 300, (rows, kv, dim), generator=gen).float() / 2)
    v[0, 0, :6] = torch.tensor([float("nan"), float("inf"), -float("inf"), 127.5, -128.5, 0.5])
    scale = torch.tensor([1.0, 0.25])
    s = rotation(1, rows, kv, kv, dim, 0, F32, weight=None)
    k_scale = torch.ones(kv)
    cache = [torch.zeros((1, rows, kv, dim), dtype=I8, device=DEV) for _ in range(2)]
    q = s["q"].clone()
    got = A.norm_rotate_append(ctx, q, s["k"], v.to(DEV), torch.arange(rows, device=DEV), cache[0], cache[1], s["positions"],
                               s["cos"], s["sin"], None, None, EPS, k_scale=k_scale.to(DEV), v_scale=scale.to(DEV), out=q)
    assert got is q
    plan = EN.encode([rows, kv, dim], "float32", [EN.Quantize(EN.BindingParam("scale", "float32", (kv,)), axis=1)])
    b = P.Bound(P.Plan(plan.blob), {}, {"scale": ("float32", [kv], scale.numpy().tobytes())})
    out = torch.empty((rows, kv, dim), dtype=I8, device=DEV)
    x = v.to(DEV)
    torch.cuda.synchronize()
    ctx.relayout_device(b, x.data_ptr(), out.data_ptr())
    ctx.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(cache[1][0], out)
    check_rotated(q, s["q"], None, s, 0, False, "q in place")


# ------------------------------------------------------------ attention

def attend(ctx, s, lse=True, **more):
    d = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    # the order in memory goes with .to() for dense transposes; keep it for sure
    for x in ("cache_k", "cache_v"):
        if not s[x].is_contiguous():
            d[x] = s[x].transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    out_lse = torch.full(s["q"].shape[:2], 7.0, device=DEV) if lse else None
    out = A.tree_attention(ctx, d["q"], d["cache_k"], d["cache_v"], d["table"], d["cached"], d["starts"], mask=d["mask"],
                           scale=d["scale"], k_scale=d["k_scale"], v_scale=d["v_scale"], lse=out_lse, **more)
    torch.cuda.synchronize()
    return out, out_lse


def check_attention(ctx, s, what, **more):
    say("attend", what)
    out, lse = attend(ctx, s, **more)
    want, want_lse, bound = C.attention(s["q"], s["cache_k"], s["cache_v"], s["table"], s["cached"], s["starts"], s["mask"],
                                        s["scale"], s["k_scale"], s["v_scale"], s["q"].dtype)
    u = 2.0 ** -24 if s["q"].dtype == F16 else 0.0
    within(out, want, bound + u, what)
    empty = torch.isinf(want_lse)
    got = lse.double().cpu()
    assert torch.equal(torch.isinf(got), empty)
    # the sum's own error, and 2^-21 of the maximum that is added back
    assert bool(((got - want_lse)[~empty].abs() <= 2.0 ** -17 * (1 + want_lse[~empty].abs())).all()), what
    return out


SIZES = [
    # heads, kv, dim, page, order
    (8, 2, 128, 16, "slots"), (8, 8, 128, 64, "heads"), (4, 1, 64, 16, "slots"), (6, 2, 80, 16, "slots"),
    (3, 3, 64, 24, "heads"), (6, 1, 256, 32, "heads"), (4, 2, 136, 16, "slots"), (24, 2, 40, 5, "slots"), (16, 1, 128, 1, "heads"),
    (2, 1, 8, 8, "slots"), (5, 1, 200, 48, "slots")]


@pytest.mark.parametrize("heads,kv,dim,page,order", SIZES)
@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, I8), (BF16, I8)])
def test_tree_attention_sizes(ctx, heads, kv, dim, page, order, dtype, cache):
    for n, (cached, fresh, words) in enumerate([([70, 0, 33, 5], [1, 1, 1, 1], 0), ([3, 140, 31], [7, 5, 12], 1),
                                                ([64, 17], [40, 21], 0)]):
        s = C.attention_case(n + dim, cached, fresh, heads, kv, dim, dtype, cache, page, order, words)
        check_attention(ctx, s, (heads, kv, dim, page, order, dtype, cache, n))


@pytest.mark.parametrize("cached,fresh,words", [
    ([0], [1], 0), ([1], [1], 0), ([127], [1], 0), ([128], [1], 0), ([129], [1], 1), ([5000], [1], 0), ([5000], [13], 1),
    ([0, 300, 0, 9], [0, 3, 0, 2], 0), ([0, 0], [64, 70], 2), ([31, 1000], [130, 2], 3), ([77], [200], 4), ([100], [100], 1),
    ([40] * 300, [1] * 300, 0), ([0] * 70, [2] * 70, 1), ([900], [33], 0), ([2000, 3, 700, 90], [9, 17, 33, 1], 1)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_tree_attention_lengths(ctx, cached, fresh, words, dtype):
    s = C.attention_case(len(cached) + fresh[0], cached, fresh, 4, 2, 128, dtype, dtype, 16, "slots", words)
    check_attention(ctx, s, (len(cached), cached[:4], fresh[:4], words, dtype))


@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_tree_attention_leaves_out_what_no_row_sees(ctx, page, dtype):
    """NaN and infinities past the lengths, in pages of nobody, and in tokens
    that only some rows see; rows that see nothing; the result's bits are those
    without them."""
    cached, fresh = [50, 0, 200], [12, 9, 40]
    s = C.attention_case(page, cached, fresh, 6, 2, 128, dtype, dtype, page, "slots", 1)
    s["mask"][3] = 0          # sees the context alone
    s["mask"][12 + 4] = 0     # no context: nothing
    clean = check_attention(ctx, s, ("clean", page))
    for x in ("cache_k", "cache_v"):
        dirty = torch.full_like(s[x], float("nan"))
        for b, n in enumerate(c + f for c, f in zip(cached, fresh)):
            for i in range(n):
                g, o = int(s["table"][b, i // page]), i % page
                dirty[g, o] = s[x][g, o]
        s[x] = dirty
    out, _ = attend(ctx, s)
    assert torch.equal(out, clean)
    # one token of request 2 that only itself and its descendants see
    g, o = divmod(200 + 17, page)
    g = int(s["table"][2, g])
    s["cache_v"][g, o, 0, 5], s["cache_v"][g, o, 1, 9] = float("inf"), float("nan")
    out, _ = attend(ctx, s)
    sees = torch.zeros(61, dtype=torch.bool)
    for r in range(21, 61):
        sees[r] = bool(int(s["mask"][r, 0]) >> 17 & 1)
    assert 0 < int(sees.sum()) < 40
    assert torch.equal(out[~sees], clean[~sees])
    assert torch.isinf(out[sees][:, :3, 5]).all() and torch.isnan(out[sees][:, 3:, 9]).all()
    s["cache_k"][g, o] = -float("inf")  # and its keys: rows that do not see it stay
    out, _ = attend(ctx, s)
    assert torch.equal(out[~sees], clean[~sees])


@pytest.mark.parametrize("page", [16, 20])
def test_tree_attention_leaves_out_pages_that_are_none(ctx, page):
    s = C.attention_case(page, [100, 90], [3, 4], 4, 2, 64, F16, F16, page)
    s["table"][0, 2], s["table"][1, 0], s["table"][1, 3] = -1, s["cache_k"].shape[0], 1 << 30
    check_attention(ctx, s, ("pages", page))
    s["table"][:] = -1
    out, lse = attend(ctx, s)
    assert not out.any() and torch.isinf(lse).all()


def test_tree_attention_rows_of_no_request_and_empty_calls(ctx):
    s = C.attention_case(1, [20, 9], [5, 6], 4, 2, 64, BF16, BF16, 16)
    s["starts"] = torch.tensor([2, 6, 9], dtype=torch.int32)  # rows 0, 1, 9, 10 belong to nobody
    check_attention(ctx, s, "rows of no request")
    s["starts"] = torch.tensor([0, 4, 40], dtype=torch.int32)  # beyond the rows: as far as they go
    clip = dict(s, starts=torch.tensor([0, 4, 11], dtype=torch.int32))
    assert torch.equal(attend(ctx, s)[0], attend(ctx, clip)[0])
    none = dict(s, q=s["q"][:0], starts=torch.zeros(3, dtype=torch.int32))
    assert attend(ctx, none)[0].shape == (0, 4, 64)
    empty = dict(s, cache_k=s["cache_k"][:0], cache_v=s["cache_v"][:0])
    out, lse = attend(ctx, empty)
    assert not out.any() and torch.isinf(lse).all()
    narrow = C.attention_case(2, [20, 60], [5, 6], 4, 2, 64, BF16, BF16, 16, columns=3)
    check_attention(ctx, narrow, "lengths past the table")


def test_tree_attention_of_large_scores_and_equal_ones(ctx):
    """Scores far apart (a weight of one), and keys of zero (equal weights)."""
    for dtype in (F16, BF16):
        s = C.attention_case(4, [300, 40], [5, 9], 4, 2, 128, dtype, dtype, 16, tree_words=1, std=5.0)
        check_attention(ctx, s, ("large", dtype))
        s["cache_k"].zero_()
        check_attention(ctx, s, ("equal", dtype))
        s = C.attention_case(4, [3000], [2], 4, 2, 64, dtype, dtype, 16)
        s["cache_k"][int(s["table"][0, 100]), 3] *= 30  # one token far above thousands of small ones
        check_attention(ctx, s, ("outlier", dtype))


def test_tree_attention_is_the_same_every_time(ctx):
    """Twice alike, whatever the workspace holds, and into a strided result."""
    s = C.attention_case(6, [1500, 700], [20, 30], 8, 2, 128, F16, F16, 16, tree_words=1)
    first, lse = attend(ctx, s)
    room = torch.full((A.tree_attention_workspace(50, 2, 8, 2, 128, 16),), 0xff, dtype=torch.uint8, device=DEV)
    out = torch.zeros((50, 3, 8, 130), dtype=F16, device=DEV)
    again, lse2 = attend(ctx, s, workspace=room, out=out[:, 1, :, :128])
    assert torch.equal(first, again) and torch.equal(lse, lse2)
    assert not out[:, 0].any() and not out[:, 2].any() and not out[..., 128:].any()


def test_tree_attention_past_four_gigabytes(ctx):
    """A cache whose last pages lie beyond 2^32 bytes."""
    say("past 4 GiB")
    kv, dim, page = 8, 128, 64
    pages = (1 << 32) // (kv * dim * page) + 40
    keys = torch.zeros((pages, page, kv, dim), dtype=I8, device=DEV)
    values = torch.zeros((pages, page, kv, dim), dtype=I8, device=DEV)
    s = C.attention_case(3, [300, 90], [3, 4], 8, kv, dim, F16, I8, page)
    n = s["cache_k"].shape[0]
    keys[-n:], values[-n:] = s["cache_k"].to(DEV), s["cache_v"].to(DEV)
    near = attend(ctx, s)[0]
    t = s["table"].to(DEV)
    far = A.tree_attention(ctx, s["q"].to(DEV), keys, values, torch.where(t >= 0, t + (pages - n), t), s["cached"].to(DEV),
                           s["starts"].to(DEV), scale=s["scale"], k_scale=s["k_scale"].to(DEV), v_scale=s["v_scale"].to(DEV))
    assert torch.equal(near, far)
    r = rotation(2, 3, 8, kv, dim, dim, F16)
    slots = torch.tensor([pages * page - 1, pages * page - 70, 5], device=DEV)
    A.norm_rotate_append(ctx, r["q"], r["k"], r["k"], slots, keys, values, r["positions"], r["cos"], r["sin"], None, None, EPS,
                         k_scale=torch.full((kv,), 0.02, device=DEV), v_scale=torch.full((kv,), 0.02, device=DEV))
    torch.cuda.synchronize()
    want = (r["k"].float() * torch.tensor(1 / 0.02)).round().clamp(-128, 127)
    assert (values.view(-1, kv, dim)[slots].float() - want).abs().max() <= 1


# --------------------------------------------------- streams, graphs, a step

def step(ctx, s, out):
    """The four calls of a serving step into the state's own buffers."""
    t = A.block_tables(ctx, s["cached"], s["fresh"], s["table"], s["free"], s["page"], s["q"].shape[0], parents=s["parents"],
                       out=s["tables"])
    q = A.norm_rotate_append(ctx, s["q"], s["k"], s["v"], t.slots, s["cache_k"], s["cache_v"], t.positions, s["cos"], s["sin"],
                             s["qw"], s["kw"], EPS, out=s["zq"])
    return A.tree_attention(ctx, q, s["cache_k"], s["cache_v"], s["table"], s["cached"], t.starts, mask=t.mask, out=out,
                            workspace=s["room"])


def step_state(seed):
    import random
    rng = random.Random(seed)
    gen = torch.Generator().manual_seed(seed)
    cached, fresh, page, heads, kv, dim = [40, 0, 333], [7, 3, 12], 16, 8, 2, 64
    rows = sum(fresh)
    table = torch.full((3, 24), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(cached):
        n = -(-c // page)
        table[b, :n] = torch.arange(at, at + n)
        at += n
    s = dict(cached=torch.tensor(cached, dtype=torch.int32), fresh=torch.tensor(fresh, dtype=torch.int32), table=table,
             free=torch.arange(at, at + 6, dtype=torch.int32), qw=torch.rand(dim, generator=gen).to(F16),
             kw=torch.rand(dim, generator=gen).to(F16),
             parents=torch.tensor([p for n in fresh for p in C.tree(rng, n)], dtype=torch.int32))
    a = torch.rand((400, dim // 2), generator=gen) * 6
    s.update(cos=a.cos(), sin=a.sin(), q=torch.randn((rows, heads, dim), generator=gen).to(F16))
    s.update(k=torch.randn((rows, kv, dim), generator=gen).to(F16), v=torch.randn((rows, kv, dim), generator=gen).to(F16))
    for x in ("cache_k", "cache_v"):
        s[x] = torch.randn((at + 6, page, kv, dim), generator=gen).to(F16)
    s = {k: v.to(DEV) for k, v in s.items()}
    i32 = dict(dtype=torch.int32, device=DEV)
    s.update(page=page, zq=torch.empty_like(s["q"]), tables=A.Tables(
        torch.empty(4, **i32), torch.empty(rows, dtype=torch.int64, device=DEV), torch.empty(rows, **i32),
        torch.empty(1, **i32), torch.empty((rows, 1), dtype=torch.int64, device=DEV)),
        room=torch.empty(A.tree_attention_workspace(rows, 3, heads, kv, dim, page), dtype=torch.uint8, device=DEV))
    return s


def test_a_step_attends_over_what_it_appended(ctx):
    say("step")
    s = step_state(1)
    out = step(ctx, s, torch.empty_like(s["q"]))
    torch.cuda.synchronize()
    want, _, bound = C.attention(s["zq"].cpu(), s["cache_k"].cpu(), s["cache_v"].cpu(), s["table"].cpu(), s["cached"].cpu(),
                                 s["tables"].starts.cpu(), s["tables"].mask.cpu(), 64 ** -0.5, None, None, F16)
    within(out, want, bound + 2.0 ** -24, "step")


def test_on_another_stream_after_its_producers(ctx):
    say("streams")
    s = step_state(2)
    want = step(ctx, s, torch.empty_like(s["q"])).clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    src = s["q"].clone()
    for _ in range(5):
        s["q"].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(2_000_000)
            s["q"].copy_(src)
            out = step(ctx, s, torch.empty_like(src))
        side.synchronize()
        assert torch.equal(out, want)


def test_in_a_graph(ctx):
    """Captured once, replayed with other inputs between the program's own work."""
    say("graph")
    s = step_state(3)
    out = torch.empty_like(s["q"])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(ctx, s, out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(ctx, s, out)
    gen = torch.Generator(device=DEV).manual_seed(1)
    for _ in range(4):
        s["q"].copy_(torch.randn(s["q"].shape, generator=gen, device=DEV))
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        eager = step(ctx, s, torch.empty_like(out))
        torch.cuda.synchronize()
        assert torch.equal(got, eager)


def test_over_the_cache_of_a_plan(ctx):
    """The C5 plan's int8 result [B, heads, S, dim], made on the GPU, is a cache
    of one page a request."""
    say("plan's cache")
    from sym_amd import workloads as W
    b, n = 2, 48
    made = []
    for seed in (1, 2):
        x, sc = W.c5_input(b, n, heads=4, dim=64, seed=seed)
        bound = P.Bound(P.Plan(W.c5_plan(4, 64).blob), {"B": b, "S": n}, W.param("scale", sc))
        out = torch.empty((b, 4, n, 64), dtype=I8, device=DEV)
        ctx.execute_h2d(bound, x.ctypes.data, x.nbytes, out.data_ptr(), out.numel())
        made.append((out, torch.from_numpy(sc)))
    gen = torch.Generator().manual_seed(3)
    s = dict(q=torch.randn((2, 8, 64), generator=gen).to(F16), cache_k=made[0][0].cpu().transpose(1, 2),
             cache_v=made[1][0].cpu().transpose(1, 2), table=torch.tensor([[0], [1]], dtype=torch.int32),
             cached=torch.tensor([n - 1, n - 1], dtype=torch.int32), starts=torch.tensor([0, 1, 2], dtype=torch.int32),
             mask=None, k_scale=made[0][1], v_scale=made[1][1], scale=64 ** -0.5)
    check_attention(ctx, s, "plan's cache")


# ------------------------------------------------------------ refusals

def test_refusals(ctx):
    say("refusals")
    s = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v
         for k, v in C.attention_case(1, [20], [2], 4, 2, 64, F16, F16, 16, tree_words=1).items()}

    def go(**more):
        d = dict(s, **more)
        return A.tree_attention(ctx, d["q"], d["cache_k"], d["cache_v"], d["table"], d["cached"], d["starts"],
                                mask=d["mask"], k_scale=d["k_scale"], v_scale=d["v_scale"], workspace=d.get("room"))

    go()
    for bad in (dict(q=s["q"].float()), dict(q=s["q"].to(BF16)), dict(q=s["q"].cpu()), dict(q=s["q"][:, :3]),
                dict(cache_v=s["cache_v"][:1]), dict(cache_k=s["cache_k"].float(), cache_v=s["cache_v"].float()),
                dict(k_scale=torch.ones(2, device=DEV)), dict(cache_k=s["cache_k"].to(I8), cache_v=s["cache_v"].to(I8)),
                dict(table=s["table"].long()), dict(cached=s["cached"].long()), dict(starts=s["starts"][:1]),
                dict(mask=s["mask"][:1]), dict(mask=s["mask"].int()),
                dict(cache_k=s["cache_k"].transpose(2, 3).contiguous().transpose(2, 3))):
        with pytest.raises(ValueError):
            go(**bad)
    with pytest.raises(P.TransferError, match="insufficient_capacity"):
        go(room=torch.empty(64, dtype=torch.uint8, device=DEV))
    odd = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v
           for k, v in C.attention_case(1, [20], [2], 4, 2, 60, F16, F16, 16).items()}
    with pytest.raises(P.TransferError, match="unsupported_layout"):
        go(**odd)
    r = rotation(1, 4, 2, 1, 64, 64, F16)
    args = [r["q"], r["k"], r["positions"], r["cos"], r["sin"], r["q_weight"], r["k_weight"], EPS]
    for i, bad in ((1, r["k"][:3]), (1, r["k"].float()), (2, r["positions"].long()), (3, r["cos"][:, :3]),
                   (5, r["q_weight"][:5]), (6, r["k_weight"].to(F16)), (0, r["q"].cpu())):
        with pytest.raises(ValueError):
            A.norm_rotate(ctx, *(args[:i] + [bad] + args[i + 1:]))
    wide = torch.zeros((97, 40), device=DEV)
    with pytest.raises(P.TransferError, match="invalid_argument"):
        A.norm_rotate(ctx, *(args[:3] + [wide, wide] + args[5:]))
    big = torch.zeros((1, 1, 520), dtype=F16, device=DEV)
    with pytest.raises(P.TransferError, match="unsupported_layout"):
        A.norm_rotate(ctx, big, big, r["positions"][:1], r["cos"], r["sin"], None, None, EPS)
    i32 = torch.zeros(2, dtype=torch.int32, device=DEV)
    table = torch.zeros((2, 4), dtype=torch.int32, device=DEV)
    for bad in (dict(page=0), dict(rows=-1), dict(cached=i32[:1]), dict(fresh=i32.long()), dict(parents=i32)):
        d = dict(dict(cached=i32, fresh=i32, page=16, rows=5, parents=None), **bad)
        with pytest.raises(ValueError):
            A.block_tables(ctx, d["cached"], d["fresh"], table, i32, d["page"], d["rows"], parents=d["parents"])
    closed = P.Context(0)
    closed.close()
    with pytest.raises((P.TransferError, ValueError)):
        A.block_tables(closed, i32, i32, table, i32, 16, 0)
