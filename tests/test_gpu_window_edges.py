"""Attention over packed sequences and its gradients, on the GPU: buffers that calls
share, numbers of first tokens, gradients that lie anyhow,
sequences shorter and longer than the window."""
import pytest

from tests import window_cases as W
from tests.test_gpu_window import check

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
