"""Attention over packed sequences and its gradients, on the GPU: buffers that calls
share, numbers of first tokens, gradients that lie anyhow, sequences shorter and longer
than the window, forms of large batches, places around operands and results."""
import ctypes

import pytest

from tests import window_cases as W
from tests.test_gpu_window import check, within

torch = pytest.importorskip("torch")
from sym_amd import _native as N  # noqa: E402
from sym_amd import attention as A  # noqa: E402
from sym_amd import pyreloc as P  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16
NAN = float("nan")


@pytest.fixture(scope="module")
def ctx():
    c = P.Context(0)
    yield c
    c.close()


def say(*what):
    print(*what, flush=True)


def packed(seed, lengths, heads, kv, dim, dtype):
    s = W.window_case(seed, lengths, heads, kv, dim, dtype, fused=False)
    return [s[n].to(DEV) for n in "qkv"], s["starts"].to(DEV), s["dout"].to(DEV)


def test_one_lse_buffer_for_two_calls(ctx):
    """A program may keep one buffer for all layers: each backward has its own numbers."""
    say("one lse buffer")
    buffer = torch.empty((4, 160), device=DEV)
    layers = [packed(31 + i, [100, 60], 4, 2, 64, BF16) for i in range(2)]
    outs = []
    for qkv, starts, dout in layers:
        leaves = [t.requires_grad_() for t in qkv]
        out = A.window_attention(ctx, *leaves, starts, window=30, sinks=2, lse=buffer)
        own = A.window_attention(ctx, *leaves, starts, window=30, sinks=2)
        kept = torch.empty_like(buffer)
        A.window_attention(ctx, *(t.detach() for t in leaves), starts, window=30, sinks=2, lse=kept)
        assert torch.equal(buffer, kept)  # the caller's is filled all the same
        outs.append((out, own, leaves, dout))
    for out, own, leaves, dout in outs:
        for x, y in zip(torch.autograd.grad(out, leaves, dout), torch.autograd.grad(own, leaves, dout)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("sinks", [257, 1000])
def test_first_tokens_that_every_window_holds(ctx, sinks):
    """However many, where no row leaves the window."""
    check(ctx, W.window_case(34, [90, 40], 2, 1, 64, BF16), "first tokens", 130, sinks)


def test_gradients_that_lie_anyhow(ctx):
    """A result's gradient at an address of no 16 bytes, or with rows that no kernel steps over."""
    say("gradients that lie anyhow")
    qkv, starts, dout = packed(33, [70, 33], 4, 2, 64, F16)
    leaves = [t.requires_grad_() for t in qkv]
    out = A.window_attention(ctx, *leaves, starts, window=25, sinks=1)
    want = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    room = torch.zeros(dout.numel() + 1, dtype=F16, device=DEV)
    room[1:] = dout.flatten()
    wide = torch.zeros((103, 4, 65), dtype=F16, device=DEV)
    wide[..., :64] = dout
    for given in (room[1:].view(dout.shape), wide[..., :64], dout.transpose(0, 2).contiguous().transpose(0, 2)):
        assert torch.equal(given, dout)
        for x, y in zip(torch.autograd.grad(out, leaves, given, retain_graph=True), want):
            assert torch.equal(x, y)
    # as it comes about: a result beside another tensor of an odd length
    both = torch.cat([torch.zeros(1, dtype=F16, device=DEV), out.flatten()])
    weights = torch.cat([torch.zeros(1, dtype=F16, device=DEV), dout.flatten()])
    for x, y in zip(torch.autograd.grad(both, leaves, weights), want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16)])
def test_short_and_long_sequences_with_first_tokens(ctx, dim, dtype):
    """Those that no window leaves have no sums of first tokens; the others keep theirs apart."""
    lengths = [30, 0, 41, 200, 12, 40, 42, 170, 1, 300, 39, 43, 500, 5, 45, 45, 45]
    check(ctx, W.window_case(36, lengths, 4, 2, dim, dtype, before=50, after=70), "short and long", 40, 33)
    check(ctx, W.window_case(37, lengths, 2, 2, dim, dtype, before=3), "a narrow window", 2, 5)


@pytest.mark.parametrize("heads,kv,dim,dtype", [(8, 8, 64, F16), (16, 16, 128, BF16)])
def test_a_long_sequence_of_many_first_tokens(ctx, heads, kv, dim, dtype):
    """Pieces of rows longer than the least, and no power of two; D of the result alone."""
    blocks = 8
    assert 2100 * kv * blocks // 768 > 128 and (2100 * kv * blocks // 768 + 31) // 32 in (6, 11)
    check(ctx, W.window_case(35, [2100], heads, kv, dim, dtype), "long, many first tokens", 300, 256)


@pytest.mark.parametrize("starts", [[-5, 100, 10 ** 9], [50, 20, 160], [160, 0], [2 ** 31 - 1, -2 ** 31], [0, 60, 160]])
def test_nothing_outside_the_operands(ctx, starts):
    """Starts out of order or out of range: what lies around results and workspace stays, and
    what lies around operands reaches nothing."""
    say("nothing outside", starts)
    rows, heads, kv, dim, pad = 160, 4, 2, 64, 4096
    s = W.window_case(38, [100, 60], heads, kv, dim, BF16, fused=False)

    def put(t, around):  # inside a larger buffer
        room = torch.full((t.numel() + 2 * pad,), around, dtype=t.dtype, device=DEV)
        room[pad:-pad] = t.to(DEV).flatten()
        return room, room[pad:-pad].view(t.shape)
    q, k, v, dout = (put(s[n], NAN)[1] for n in ("q", "k", "v", "dout"))
    made = {n: put(t, 7.0) for n, t in dict(out=torch.zeros_like(s["q"]), lse=torch.zeros((heads, rows)), dq=torch.zeros_like(s["q"]),
                                            dk=torch.zeros_like(s["k"]), dv=torch.zeros_like(s["v"])).items()}
    z = torch.tensor(starts, dtype=torch.int32, device=DEV)
    out, lse = made["out"][1], made["lse"][1]
    A.window_attention(ctx, q, k, v, z, window=30, sinks=40, out=out, lse=lse)
    args, device = A._window_record(ctx, q, k, v, out, lse, z, 30, 40, None)
    size, err = ctypes.c_size_t(), N.relx_err()
    assert N.lib().relx_window_attention_workspace(args, ctypes.byref(size), ctypes.byref(err)) == 0
    room, workspace = put(torch.zeros(size.value // 4), 7.0)
    A._call("relx_window_attention_backward", ctx, args, A._heads(dout, "", dout.shape, BF16, device),
            *(A._heads(made[n][1], "", made[n][1].shape, BF16, device) for n in ("dq", "dk", "dv")), workspace.data_ptr(),
            size.value, A._stream(device))
    torch.cuda.synchronize()
    for name, (whole, inside) in dict(made, workspace=(room, workspace)).items():
        assert (whole[:pad] == 7.0).all() and (whole[-pad:] == 7.0).all(), name
    for name in ("out", "dq", "dk", "dv"):
        assert torch.isfinite(made[name][1]).all(), name
    if starts == [0, 60, 160]:
        want = W.window_attention(s["q"], s["k"], s["v"], torch.tensor(starts), 30, 40, dim ** -0.5, s["dout"])
        for name, x in (("out", "o"), ("dq", "dq"), ("dk", "dk"), ("dv", "dv")):
            within(made[name][1], want[x], want["b" + x], name)


@pytest.mark.parametrize("dtype,dim", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("lengths,window,sinks", [([2100], None, 0), ([30, 2500, 2100], 1000, 4)])
def test_rows_that_see_few_tokens(ctx, dtype, dim, lengths, window, sinks):
    """In long sequences too their D is summed in 32 bits: where values have much in common,
    dP and D are large beside their difference, and D of the rounded result would be off by
    more than all of the bound."""
    say("few tokens", lengths)
    heads, kv, scale = 2, 1, dim ** -0.5
    s = W.window_case(39, lengths, heads, kv, dim, dtype, fused=False, std=0.25)
    s["v"] = (8 + s["v"].float()).to(dtype)
    s["dout"] = (1 + s["dout"].float()).to(dtype)
    leaves = [s[n].to(DEV).requires_grad_() for n in "qkv"]
    out = A.window_attention(ctx, *leaves, s["starts"].to(DEV), window=window, sinks=sinks)
    dq = torch.autograd.grad(out, leaves[0], s["dout"].to(DEV))[0].cpu().double()
    u, f32 = W.ROUND[dtype], W.F32
    for a, b in zip(s["starts"].tolist(), s["starts"].tolist()[1:]):
        n = min(b - a, 128)  # rows that see up to so many
        see = W.sees(n, window, sinks)
        for h in range(heads):
            q, k, v, do = (s[x][a:a + n, y].double() for x, y in (("q", h), ("k", 0), ("v", 0), ("dout", h)))
            p = torch.softmax(torch.where(see, q @ k.T * scale, -float("inf")), 1)
            dp, size = do @ v.T, do.abs() @ v.abs().T
            g = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
            # scores and lse in 32 bits: weights off by 2 ds; dP, its products with them and
            # their sum: in 32 bits; dS rounded to u of itself (f16: or 2^-30 of the largest)
            ds = (dim + 4) * f32 * (q.abs() @ k.abs().T * see).amax(1, keepdim=True) * scale + 8 * f32 * (1 + n) ** 0.5
            d_off = (2 * ds + (dim + n + 8) * f32) * (p * size).sum(1, keepdim=True)
            off = u * g.abs() + p * scale * ((2 * ds + (dim + 8) * f32) * size + d_off) + see * 2.0 ** -30 * scale * float(size.max())
            want = g @ k
            bound = (off + (n / 32 + 16) * f32 * g.abs()) @ k.abs() + u * want.abs() + W.STEP[dtype]
            far = (dq[a:a + n, h] - want).abs() - bound
            assert float(far.max()) <= 0, (a, h, float(far.max()))
