"""Attention over packed sequences and its gradients, on the GPU: buffers that calls
share, numbers of first tokens."""
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
