"""Attention over packed sequences with a window and first tokens that stay, and
its gradients, on the GPU."""
import pytest

from tests import window_cases as W

torch = pytest.importorskip("torch")
from sym_amd import attention as A  # noqa: E402
from sym_amd import pyreloc as P  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ctx():
    c = P.Context(0)
    yield c
    c.close()


def say(*what):
    print(*what, flush=True)


def within(got, want, bound, what):
    off = (got.cpu().double() - want).abs() - bound
    assert not torch.isnan(off).any(), what
    assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()))


def check(ctx, s, what, window=None, sinks=0, scale=None, back=True):
    say(what, [int(x) for x in s["starts"]], list(s["q"].shape), list(s["k"].shape), window, sinks)
    dim = s["q"].shape[2]
    want = W.window_attention(s["q"], s["k"], s["v"], s["starts"], window, sinks, dim ** -0.5 if scale is None else scale,
                              s["dout"] if back else None)
    whole = torch.cat([s["q"], s["k"], s["v"]], 1).to(DEV)  # views of one tensor
    q, k, v = whole.split([s[n].shape[1] for n in "qkv"], 1)
    starts, dout = s["starts"].to(DEV), s["dout"].to(DEV)
    lse = torch.full((q.shape[1], q.shape[0]), 7.0, device=DEV)
    see = dict(window=window, sinks=sinks, scale=scale)
    out = A.window_attention(ctx, q, k, v, starts, lse=lse, **see)
    within(out, want["o"], want["bo"], (what, "out"))
    assert torch.equal(lse.cpu() == -float("inf"), want["lse"] == -float("inf")), what
    real = want["lse"] > -float("inf")
    off = (lse.cpu().double() - want["lse"]).abs() - (want["ds"] + 4e-6 * (1 + want["lse"].abs()))
    assert not real.any() or float(off[real].max()) <= 0, (what, "lse")
    if not back:
        return
    got = A.window_attention_backward(ctx, dout, q, k, v, out, lse, starts, **see)
    for name, g in zip(("dq", "dk", "dv"), got):
        within(g, want[name], want["b" + name], (what, name))
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = A.window_attention(ctx, *leaves, starts, **see)
    assert torch.equal(o.detach(), out)
    for g, h in zip(got, torch.autograd.grad(o, leaves, dout)):
        assert torch.equal(g, h), what  # the same bits every time


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lengths,heads,kv,dim,window,sinks", [
    ([1], 1, 1, 64, None, 0),
    ([5], 2, 1, 128, None, 0),
    ([64], 1, 1, 64, 16, 1),
    ([200], 4, 2, 128, None, 0),
    ([200], 4, 1, 128, 64, 4),
    ([333, 0, 17, 128], 6, 2, 80, 100, 1),
    ([130, 300], 3, 1, 96, 33, 40),
    ([257], 8, 8, 64, 1, 0),
    ([257], 2, 1, 72, 1, 3),
    ([500], 16, 2, 128, 129, 17),
    ([90, 41], 20, 1, 64, 30, 2),
    ([70], 40, 2, 8, 5, 70),
    ([700], 2, 2, 128, 300, 256),
    ([300], 2, 1, 64, 10 ** 12, 256),
])
def test_results_and_gradients(ctx, dtype, lengths, heads, kv, dim, window, sinks):
    check(ctx, W.window_case(1, lengths, heads, kv, dim, dtype), str(dtype), window, sinks)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_many_sequences(ctx, dtype):
    check(ctx, W.window_case(2, W.ragged(3, 150, 40), 2, 1, 64, dtype), "many", 9, 2)


def test_long_sequences(ctx):
    """Several pieces of rows add to the first tokens' gradients."""
    check(ctx, W.window_case(3, [1500, 40, 1100], 2, 1, 64, BF16), "long", 70, 5)
    check(ctx, W.window_case(4, [1300], 1, 1, 128, F16), "long", 200, 40)


@pytest.mark.parametrize("dtype,kv,lengths,dim", [(BF16, 43, [700], 128), (F16, 90, [300, 130], 128), (BF16, 86, [15] * 12, 64),
                                                  (F16, 172, [200, 90, 130], 64)])
def test_many_keys(ctx, dtype, kv, lengths, dim):
    """Enough tiles of keys for the form of large batches."""
    assert (sum(lengths) // 128 + len(lengths)) * kv >= (256 if dim > 64 else 1024)
    check(ctx, W.window_case(15, lengths, kv, kv, dim, dtype), "many keys", 60, 5)


def test_rows_of_no_sequence(ctx):
    s = W.window_case(5, [100, 50], 4, 2, 64, BF16, before=37, after=150)
    check(ctx, s, "padded", 40, 2)
    # whatever those rows hold, and what other sequences do
    for n in ("q", "k", "v", "dout"):
        s[n] = s[n].clone()
    outs = []
    for bad in (0.0, float("nan")):
        t = {n: s[n].clone() for n in ("q", "k", "v", "dout")}
        for x in t.values():
            x[:37], x[187:] = bad, bad
            x[137:187] = bad if bad else x[137:187]
        leaves = [t[n].to(DEV).requires_grad_() for n in "qkv"]
        o = A.window_attention(ctx, *leaves, s["starts"].to(DEV), window=40, sinks=2)
        outs.append([o.detach(), *torch.autograd.grad(o, leaves, t["dout"].to(DEV))])
    for x, y in zip(*outs):
        assert torch.equal(x[:137], y[:137]) and torch.equal(x[187:], y[187:])
        assert not y[:37].any() and not y[187:].any()
        assert torch.isnan(y[137:187]).any()
    empty = torch.zeros((0, 4, 64), dtype=BF16, device=DEV)
    z = torch.zeros(3, dtype=torch.int32, device=DEV)
    assert A.window_attention(ctx, empty, empty, empty, z).shape == (0, 4, 64)
    none = A.window_attention(ctx, *(s[n].to(DEV) for n in "qkv"), z[:1], window=3)
    assert not none.any()


def test_starts_that_do_not_fit(ctx):
    """Out of order or out of range: nothing outside the operands is read or written."""
    s = W.window_case(6, [100, 60], 2, 1, 64, BF16)
    q, k, v, do = (s[n].to(DEV) for n in ("q", "k", "v", "dout"))
    for starts in ([-5, 100, 10 ** 9], [50, 20, 160], [160, 0], [2 ** 31 - 1, -2 ** 31]):
        z = torch.tensor(starts, dtype=torch.int32, device=DEV)
        lse = torch.zeros((2, 160), device=DEV)
        o = A.window_attention(ctx, q, k, v, z, window=30, sinks=3, lse=lse)
        A.window_attention_backward(ctx, do, q, k, v, o, lse, z, window=30, sinks=3)
        torch.cuda.synchronize()


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
def test_scales(ctx, scale):
    check(ctx, W.window_case(7, [150], 2, 1, 64, F16), "scale %g" % scale, 50, 3, scale)


@pytest.mark.parametrize("size", [1e-4, 1e-2, 100.0])
def test_small_and_large_gradients_in_f16(ctx, size):
    """The gradients of scores are scaled before they are rounded."""
    s = W.window_case(8, [300], 4, 1, 128, F16)
    s["dout"] = (s["dout"].float() * size).to(F16)
    check(ctx, s, "gradients of %g" % size, 100, 4)


def test_large_scores(ctx):
    """A row's maximum is far above the others, and moves."""
    s = W.window_case(9, [400], 2, 1, 64, F16, std=6.0)
    s["dout"] = (s["dout"].float() / 6).to(F16)
    check(ctx, s, "large scores", 150, 2)


def test_gradients_against_differences(ctx):
    """Of the kernel's own results, summed against a random direction in 64 bits."""
    s = W.window_case(10, [90], 2, 1, 64, F16, std=0.5)
    leaves = [s[n].to(DEV).requires_grad_() for n in "qkv"]
    starts, dout = s["starts"].to(DEV), s["dout"].to(DEV)
    o = A.window_attention(ctx, *leaves, starts, window=20, sinks=2)
    grads = torch.autograd.grad(o, leaves, dout)
    gen = torch.Generator().manual_seed(1)
    for i in range(3):
        d = torch.randn(leaves[i].shape, generator=gen).to(DEV)
        h = 2.0 ** -4
        def value(sign):
            moved = [t.detach() for t in leaves]
            moved[i] = (moved[i].float() + sign * h * d).to(F16)
            step = moved[i].double() - leaves[i].detach().double()
            o = A.window_attention(ctx, *moved, starts, window=20, sinks=2)
            return float((o.double() * dout.double()).sum()), step
        (up, a), (down, b) = value(1), value(-1)
        slope = float((grads[i].double() * (a - b)).sum())
        # results are rounded to 2^-11 of themselves, at random, 11520 of them of size up to one
        # times gradients of size 0.5; the third derivatives' part falls with h^2
        assert abs(up - down - slope) < 4 * 2.0 ** -11 * 0.5 * 11520 ** 0.5 + 0.1 * abs(slope), (i, up - down, slope)


def test_strides(ctx):
    """Heads before rows, results into views, keys shared by broadcasting."""
    s = W.window_case(11, [70, 33], 4, 2, 64, BF16)
    starts = s["starts"].to(DEV)
    q, k, v = (s[n].to(DEV) for n in "qkv")
    want = A.window_attention(ctx, q, k, v, starts, window=25, sinks=1)
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    wide = torch.zeros((103, 8, 64), dtype=BF16, device=DEV)
    assert torch.equal(want, A.window_attention(ctx, *turned, starts, window=25, sinks=1, out=wide[:, 2:6]))
    assert torch.equal(want, wide[:, 2:6]) and not wide[:, :2].any() and not wide[:, 6:].any()
    one = k[:, :1]
    both = one.expand(103, 2, 64)
    assert torch.equal(A.window_attention(ctx, q, both.contiguous(), v, starts, window=25),
                       A.window_attention(ctx, q, both, v, starts, window=25))
    leaves = [t.detach().requires_grad_() for t in (q, one, v)]
    o = A.window_attention(ctx, leaves[0], leaves[1].expand(103, 2, 64), leaves[2], starts, window=25)
    g = torch.autograd.grad(o.sum(), leaves)  # of a gradient that is one number everywhere
    ones = torch.ones_like(o)
    leaves2 = [q.detach().requires_grad_(), both.contiguous().requires_grad_(), v.detach().requires_grad_()]
    h = torch.autograd.grad(A.window_attention(ctx, *leaves2, starts, window=25), leaves2, ones)
    assert torch.equal(g[0], h[0]) and torch.equal(g[1], h[1].sum(1, keepdim=True)) and torch.equal(g[2], h[2])


def test_other_streams_and_graphs(ctx):
    s = W.window_case(12, [200, 90], 4, 2, 128, BF16)
    starts = s["starts"].to(DEV)
    q, k, v, do = (s[n].to(DEV).contiguous() for n in ("q", "k", "v", "dout"))

    def step():
        lse = torch.empty((4, 290), device=DEV)
        o = A.window_attention(ctx, q, k, v, starts, window=60, sinks=3, lse=lse)
        return [o, *A.window_attention_backward(ctx, do, q, k, v, o, lse, starts, window=60, sinks=3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(first, step()):
        assert torch.equal(x, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = step()
    for i in range(3):
        for t in (q, k, v, do):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(made, step()):
            assert torch.equal(x, y)


def test_a_captured_training_step(ctx):
    """Forward and backward through torch's graph, replayed."""
    s = W.window_case(17, [150, 60], 4, 2, 64, BF16)
    starts = s["starts"].to(DEV)
    leaves = [s[n].to(DEV).contiguous().requires_grad_() for n in "qkv"]
    dout = s["dout"].to(DEV)

    def step():
        o = A.window_attention(ctx, *leaves, starts, window=50, sinks=2)
        return [o.detach(), *torch.autograd.grad(o, leaves, dout)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = step()
    for i in range(3):
        with torch.no_grad():
            for t in (*leaves, dout):
                t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(made, step()):
            assert torch.equal(x, y)


def test_a_training_step(ctx):
    """Norm and rotation, then attention: gradients of a fused projection and both weights against 64 bits."""
    from tests import attention_cases as C
    gen = torch.Generator().manual_seed(13)
    lengths, heads, kv, dim = [60, 100], 4, 2, 64
    rows = sum(lengths)
    fused = torch.randn((rows, heads + 2 * kv, dim), generator=gen).to(BF16)
    weights = [(1 + 0.2 * torch.randn(dim, generator=gen)).to(BF16) for _ in range(2)]
    starts = torch.tensor([0, 60, 160], dtype=torch.int32)
    positions = torch.cat([torch.arange(n) for n in lengths]).to(torch.int32)
    angle = torch.arange(100, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))
    dout = torch.randn((rows, heads, dim), generator=gen).to(BF16)
    leaf = fused.to(DEV).requires_grad_()
    w = [x.to(DEV).requires_grad_() for x in weights]
    q, k, v = leaf.split((heads, kv, kv), 1)
    q, k = A.norm_rotate(ctx, q, k, positions.to(DEV), angle.cos().float().to(DEV), angle.sin().float().to(DEV), *w, 1e-6)
    o = A.window_attention(ctx, q, k, v, starts.to(DEV), window=30, sinks=2)
    got = torch.autograd.grad(o, (leaf, *w), dout.to(DEV))
    x, wd = fused.double().requires_grad_(), [t.double().requires_grad_() for t in weights]
    at = angle[positions.long()]
    turned = [C.norm_rotate(part, z, at.cos(), at.sin(), dim, False, 1e-6)[0] for part, z in zip(x.split((heads, kv, kv), 1), wd)]
    outs = []
    for a, b in zip(starts.tolist(), starts.tolist()[1:]):
        see = W.sees(b - a, 30, 2)
        for h in range(heads):
            sc = torch.where(see, turned[0][a:b, h] @ turned[1][a:b, h // 2].T * dim ** -0.5, -float("inf"))
            outs.append(torch.softmax(sc, 1) @ x[a:b, heads + kv + h // 2])
    o64 = torch.stack([torch.cat([outs[h], outs[heads + h]]) for h in range(heads)], 1)
    want = torch.autograd.grad(o64, (x, *wd), dout.double())
    # turned queries and keys, weights of the softmax, scores' gradients, results, gradients into
    # the norm and out of it: eight roundings of 2^-9 on average, in norm
    for g, h in zip((o.detach(), *got), (o64.detach(), *want)):
        assert float((g.cpu().double() - h).norm() / h.norm()) < 8 * 2.0 ** -9


# ------------------------------------------------------------ refusals

def test_refusals(ctx):
    say("refusals")
    s = W.window_case(14, [40], 4, 2, 64, F16, fused=False)
    d = {n: s[n].to(DEV) for n in ("q", "k", "v", "starts", "dout")}
    lse = torch.empty((4, 40), device=DEV)

    def go(**more):
        x = dict(dict(d, window=8, sinks=1, lse=lse, out=None), **more)
        return A.window_attention(ctx, x["q"], x["k"], x["v"], x["starts"], window=x["window"], sinks=x["sinks"], lse=x["lse"],
                                  out=x["out"])
    out = go()
    for bad in (dict(q=d["q"].float()), dict(q=d["q"].cpu()), dict(q=d["q"][:, :3]), dict(k=d["k"].to(BF16)), dict(v=d["v"][:, :1]),
                dict(k=d["k"][:39]), dict(starts=d["starts"].long()), dict(starts=d["starts"][:0]), dict(window=-1), dict(sinks=-1),
                dict(window=None, sinks=2), dict(lse=lse.T), dict(lse=lse.half()), dict(out=out.float()),
                dict(q=d["q"].transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            go(**bad)
    for bad in (dict(sinks=257), dict(q=d["q"][..., :60], k=d["k"][..., :60], v=d["v"][..., :60]),
                dict(q=torch.zeros((40, 4, 65), dtype=F16, device=DEV)[..., :64]),
                dict(q=torch.zeros(40 * 4 * 64 + 1, dtype=F16, device=DEV)[1:].view(40, 4, 64))):
        with pytest.raises(P.TransferError, match="unsupported_layout"):
            go(**bad)
    wide = torch.zeros((40, 4, 136), dtype=F16, device=DEV)
    with pytest.raises(P.TransferError, match="unsupported_layout"):
        go(q=wide, k=wide, v=wide)
    with pytest.raises(P.TransferError, match="invalid_argument"):
        go(out=torch.zeros((40, 1, 64), dtype=F16, device=DEV).expand(40, 4, 64))
    with pytest.raises(ValueError):
        A.window_attention_backward(ctx, d["dout"], d["q"], d["k"], d["v"], out, None, d["starts"], window=8, sinks=1)
    with pytest.raises(ValueError):
        A.window_attention_backward(ctx, d["dout"].float(), d["q"], d["k"], d["v"], out, lse, d["starts"], window=8, sinks=1)
    q = d["q"].clone().requires_grad_()
    o = A.window_attention(ctx, q, d["k"], d["v"], d["starts"], window=8)
    g, = torch.autograd.grad(o.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().sum().backward()
