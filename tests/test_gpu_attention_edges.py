"""Calls of the paged-cache operators at the edges of what they take, against
their definitions (tests/attention_cases.py)."""
import pytest

from tests import attention_cases as C

torch = pytest.importorskip("torch")
from sym_amd import attention as A  # noqa: E402
from sym_amd import pyreloc as P  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32, I8 = torch.float16, torch.bfloat16, torch.float32, torch.int8


def say(*a):
    print("[gpu-case]", *a, flush=True)


@pytest.fixture(scope="module")
def ctx():
    assert torch.cuda.is_available(), "a GPU test needs the MI355X"
    c = P.Context(0)
    yield c
    c.close()


def on_gpu(s):
    return {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in s.items()}


# ------------------------------------------------------------ no requests

@pytest.mark.parametrize("dtype,cache,heads,dim,rows", [(F16, F16, 4, 64, 1), (BF16, I8, 8, 128, 9), (BF16, BF16, 6, 200, 300)])
def test_rows_without_any_request_are_zero(ctx, dtype, cache, heads, dim, rows):
    say("no requests", dtype, cache, heads, dim, rows)
    s = on_gpu(C.attention_case(1, [20], [rows], heads, 2, dim, dtype, cache, 16))
    i32 = dict(dtype=torch.int32, device=DEV)
    room = torch.full((rows, 3, heads, dim + 8), 7.0, dtype=dtype, device=DEV)
    lse = torch.full((rows, heads), 7.0, device=DEV)
    out = A.tree_attention(ctx, s["q"], s["cache_k"], s["cache_v"], torch.empty((0, 4), **i32), torch.empty(0, **i32),
                           torch.zeros(1, **i32), k_scale=s["k_scale"], v_scale=s["v_scale"], out=room[:, 1, :, :dim], lse=lse)
    torch.cuda.synchronize()
    assert not out.any() and (lse == -float("inf")).all()
    room[:, 1, :, :dim] = 7.0
    assert (room == 7.0).all()  # and nothing beside it


# ------------------------------------------------------------ no rows

@pytest.mark.parametrize("words", [1, 3])
@pytest.mark.parametrize("given", [False, True])
def test_block_tables_of_trees_without_rows(ctx, words, given):
    say("trees without rows", words)
    i32 = dict(dtype=torch.int32, device=DEV)
    out = A.Tables(torch.full((3,), -7, **i32), torch.empty(0, dtype=torch.int64, device=DEV), torch.empty(0, **i32),
                   torch.full((1,), -7, **i32), torch.empty((0, words), dtype=torch.int64, device=DEV)) if given else None
    t = A.block_tables(ctx, torch.tensor([4, 30], **i32), torch.zeros(2, **i32), torch.zeros((2, 4), **i32),
                       torch.empty(0, **i32), 16, 0, parents=torch.empty(0, **i32), words=words, out=out)
    torch.cuda.synchronize()
    assert t.starts.tolist() == [0, 0, 0] and t.taken.tolist() == [0]
    assert t.slots.shape == t.positions.shape == (0,) and t.mask.shape == (0, words)


def test_append_without_key_heads(ctx):
    """An empty cache tensor has no address either; the queries turn as ever."""
    say("append without key heads")
    gen = torch.Generator().manual_seed(1)
    q = torch.randn((3, 4, 64), generator=gen).to(F16).to(DEV)
    none, cache = torch.empty((3, 0, 64), dtype=F16, device=DEV), torch.empty((2, 16, 0, 64), dtype=F16, device=DEV)
    turn = (torch.arange(3, dtype=torch.int32, device=DEV), torch.ones((3, 32), device=DEV), torch.zeros((3, 32), device=DEV),
            None, None, 1e-6)
    out = A.norm_rotate_append(ctx, q, none, none, torch.arange(3, device=DEV), cache, cache, *turn)
    want, _ = A.norm_rotate(ctx, q, none, *turn)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# ------------------------------------------------------------ scales

# heads, kv, dim, page, cached, fresh, words: one row a key head, up to 16, 64, 128, 256
SCALED = [(4, 4, 128, 16, [70, 0, 33], [1, 1, 1], 0), (8, 2, 64, 24, [30, 3], [3, 2], 1), (8, 2, 128, 16, [40, 9], [12, 9], 1),
          (4, 2, 136, 16, [50], [20], 1), (4, 1, 128, 16, [100], [25], 0), (4, 1, 64, 32, [90], [60], 1), (2, 1, 128, 8, [33], [70], 2)]


def result(ctx, s, **more):
    d = on_gpu(s)
    lse = torch.full(s["q"].shape[:2], 7.0, device=DEV)
    out = A.tree_attention(ctx, d["q"], d["cache_k"], d["cache_v"], d["table"], d["cached"], d["starts"], mask=d["mask"],
                           scale=d["scale"], k_scale=d["k_scale"], v_scale=d["v_scale"], lse=lse, **more)
    torch.cuda.synchronize()
    return out.double().cpu(), lse.double().cpu()


def check(ctx, s, what, positive=None):
    """`positive`: the same step with a scale of zero or above, for the bound."""
    p = dict(s, **(positive or {}))
    say("attend", what)
    out, lse = result(ctx, s)
    want, want_lse, bound = C.attention(p["q"], p["cache_k"], p["cache_v"], p["table"], p["cached"], p["starts"], p["mask"],
                                        p["scale"], p["k_scale"], p["v_scale"], p["q"].dtype)
    assert not torch.isnan(out).any(), what
    assert bool(((out - want).abs() <= bound + 2.0 ** -24).all()), what
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), empty), what
    assert bool(((lse - want_lse)[~empty].abs() <= 2.0 ** -17 * (1 + want_lse[~empty].abs())).all()), what


@pytest.mark.parametrize("heads,kv,dim,page,cached,fresh,words", SCALED)
@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, I8), (BF16, I8)])
def test_tree_attention_of_scales_that_are_not_positive(ctx, heads, kv, dim, page, cached, fresh, words, dtype, cache):
    s = C.attention_case(dim + fresh[0], cached, fresh, heads, kv, dim, dtype, cache, page, tree_words=words)
    if words:
        s["mask"][1] = 0  # sees the context alone, which a request may not have
    check(ctx, dict(s, scale=0.0), ("zero", heads, kv, dim, page, dtype, cache))
    check(ctx, dict(s, scale=-0.1), ("negative", heads, kv, dim, page, dtype, cache), dict(q=-s["q"], scale=0.1))
    check(ctx, dict(s, scale=1e-30), ("tiny", heads, kv, dim, page, dtype, cache))
    if cache == I8:
        k = s["k_scale"].clone()
        k[0], k[-1] = -k[0], (0.0 if kv > 1 else -k[-1])
        check(ctx, dict(s, k_scale=k, v_scale=-s["v_scale"]), ("key scales", heads, kv, dim, page, dtype))
        check(ctx, dict(s, k_scale=k * 0), ("key scales of zero", heads, kv, dim, page, dtype))


@pytest.mark.parametrize("page", [16, 20])
@pytest.mark.parametrize("fresh", [4, 40])
def test_a_negative_scale_is_the_negative_queries_bit_for_bit(ctx, page, fresh):
    """With infinities and NaN in values that only some rows see, too."""
    s = C.attention_case(page, [50, 0], [fresh, fresh], 4, 2, 128, BF16, BF16, page, tree_words=1)
    g, o = divmod(50 + 2, page)
    s["cache_v"][int(s["table"][0, g]), o, 0, 5] = float("inf")
    s["cache_v"][int(s["table"][0, g]), o, 1, 9] = float("nan")
    out, lse = result(ctx, dict(s, scale=-0.125))
    want, want_lse = result(ctx, dict(s, q=-s["q"], scale=0.125))
    assert torch.isnan(want).any() and torch.isinf(want).any()
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out.nan_to_num(7.0), want.nan_to_num(7.0))
    assert torch.equal(lse, want_lse)


def test_a_scale_that_is_no_finite_number_is_refused(ctx):
    s = C.attention_case(1, [20], [2], 4, 2, 64, F16, F16, 16)
    for scale in (float("inf"), float("nan"), 3e38, -1e300):
        with pytest.raises(P.TransferError, match="invalid_argument"):
            result(ctx, dict(s, scale=scale))


# ------------------------------------------------------------ norms without eps

@pytest.mark.parametrize("heads,kv,dim", [(3, 1, 128), (5, 2, 64), (9, 3, 256), (1, 1, 80), (4, 4, 512)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_weight_gradients_without_eps(ctx, heads, kv, dim, dtype):
    """A wave has room for more heads than there are: what is not there adds nothing."""
    say("eps 0", heads, kv, dim, dtype)
    gen = torch.Generator().manual_seed(dim + heads)
    rows, rotary = 23, dim // 2
    x = {n: torch.randn((rows, h, dim), generator=gen).to(dtype) for n, h in (("q", heads), ("k", kv), ("dq", heads), ("dk", kv))}
    w = [(1 + 0.3 * torch.randn(dim, generator=gen)).to(dtype) for _ in range(2)]
    a = torch.rand((rows, rotary // 2), generator=gen, dtype=torch.float64) * 6
    cos, sin = a.cos().float(), a.sin().float()
    at = torch.arange(rows, dtype=torch.int32)
    d = {n: t.to(DEV) for n, t in x.items()}
    got = A.norm_rotate_backward(ctx, d["dq"], d["dk"], d["q"], d["k"], at.to(DEV), cos.to(DEV), sin.to(DEV), w[0].to(DEV),
                                 w[1].to(DEV), 0.0)
    torch.cuda.synchronize()
    u = C.ROUND[dtype]
    for i, n in enumerate("qk"):
        want, bound, want_w, size_w = C.norm_rotate_back(x["d" + n], x[n], w[i], cos.double(), sin.double(), rotary, False, 0.0)
        assert bool(((got[i].double().cpu() - want).abs() <= bound * (1 + u) + u * want.abs() + 2.0 ** -25).all()), n
        # as where eps is not zero: a term has dim / 2 + 8 roundings, its sums fewer than 192
        assert bool(((got[2 + i].double().cpu() - want_w).abs() <= (dim / 2 + 8 + 192) * C.F32 * size_w).all()), n


def test_norm_rotate_is_differentiable_once(ctx):
    say("second derivative")
    gen = torch.Generator().manual_seed(2)
    q, k = (torch.randn((3, 2, 64), generator=gen).to(DEV).requires_grad_() for _ in range(2))
    cos, sin = torch.ones((3, 32), device=DEV), torch.zeros((3, 32), device=DEV)
    at = torch.arange(3, dtype=torch.int32, device=DEV)
    zq, _ = A.norm_rotate(ctx, q, k, at, cos, sin, None, None, 1e-6)
    grad, = torch.autograd.grad((zq ** 3).sum(), q, create_graph=True)
    assert torch.isfinite(grad).all()
    with pytest.raises(RuntimeError, match="once_differentiable"):
        ((q ** 2).sum() + (grad ** 2).sum()).backward()


@pytest.mark.parametrize("wanted", [(True, False), (False, True), (False, False)])
def test_gradients_without_those_of_frozen_weights(ctx, wanted):
    say("frozen weights", wanted)
    gen = torch.Generator().manual_seed(3)
    q, k, dq, dk = (torch.randn((50, n, 80), generator=gen).to(BF16).to(DEV) for n in (5, 2, 5, 2))
    w = [torch.rand(80, generator=gen).to(BF16).to(DEV) for _ in range(2)]
    a = torch.rand((50, 40), generator=gen).to(DEV)
    args = (dq, dk, q, k, torch.arange(50, dtype=torch.int32, device=DEV), a.cos(), a.sin(), *w, 1e-6)
    every = A.norm_rotate_backward(ctx, *args)
    some = A.norm_rotate_backward(ctx, *args, weight_grads=wanted)
    torch.cuda.synchronize()
    assert torch.equal(every[0], some[0]) and torch.equal(every[1], some[1])
    for i in range(2):
        assert torch.equal(every[2 + i], some[2 + i]) if wanted[i] else some[2 + i] is None


def test_expanded_results_are_refused(ctx):
    say("expanded results")
    s = on_gpu(C.attention_case(1, [20], [3], 4, 2, 64, F16, F16, 16))
    flat = torch.zeros((1, 4, 64), dtype=F16, device=DEV)
    with pytest.raises(P.TransferError, match="invalid_argument.*overlap"):
        A.tree_attention(ctx, s["q"], s["cache_k"], s["cache_v"], s["table"], s["cached"], s["starts"], out=flat.expand(3, 4, 64))
    turn = (torch.zeros(3, dtype=torch.int32, device=DEV), torch.ones((1, 32), device=DEV), torch.zeros((1, 32), device=DEV))
    with pytest.raises(P.TransferError, match="invalid_argument.*overlap"):
        A.norm_rotate(ctx, s["q"], s["q"], *turn, None, None, 1e-6, out=(torch.empty_like(s["q"]), flat.expand(3, 4, 64)))
    k = s["q"][:, :2]
    with pytest.raises(P.TransferError, match="invalid_argument.*overlap"):
        A.norm_rotate_append(ctx, s["q"], k, k, torch.arange(3, device=DEV), s["cache_k"][:1].expand(2, 16, 2, 64),
                             s["cache_v"][:2], *turn, None, None, 1e-6)
    # reading an expanded cache is no matter
    A.tree_attention(ctx, s["q"], s["cache_k"][:1].expand(4, 16, 2, 64), s["cache_v"][:1].expand(4, 16, 2, 64), s["table"],
                     s["cached"], s["starts"])
    torch.cuda.synchronize()


@pytest.mark.parametrize("fresh,dim,cache", [(1, 128, F16), (3, 256, I8), (12, 128, F16), (12, 136, I8), (30, 64, F16), (64, 128, F16),
                                             (64, 64, I8), (100, 128, I8)])
def test_nothing_is_written_past_the_workspace(ctx, fresh, dim, cache):
    """Contexts so long that every workgroup leaves partial sums."""
    say("workspace", fresh, dim, cache)
    cached, page, heads, kv = 70_000, 64, 8, 2
    gen = torch.Generator().manual_seed(dim + fresh)
    made = [torch.randint(-9, 10, (40, page, kv, dim), generator=gen, dtype=I8).to(cache).to(DEV) for _ in range(2)]
    scale = torch.full((kv,), 0.1, device=DEV) if cache == I8 else None
    i32 = dict(dtype=torch.int32, device=DEV)
    table = torch.randint(0, 40, (1, -(-(cached + fresh) // page)), generator=gen).to(**i32)
    args = (torch.randn((fresh, heads, dim), generator=gen).to(F16).to(DEV), *made, table, torch.tensor([cached], **i32),
            torch.tensor([0, fresh], **i32))
    size = A.tree_attention_workspace(fresh, 1, heads, kv, dim, page)
    room = torch.full((size + (1 << 20),), 0xa5, dtype=torch.uint8, device=DEV)
    out = A.tree_attention(ctx, *args, k_scale=scale, v_scale=scale, workspace=room[:size])
    want = A.tree_attention(ctx, *args, k_scale=scale, v_scale=scale)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and (room[size:] == 0xa5).all() and not (room[:size] == 0xa5).all()
    with pytest.raises(P.TransferError, match="insufficient_capacity"):
        A.tree_attention(ctx, *args, k_scale=scale, v_scale=scale, workspace=room[:size - 1])
