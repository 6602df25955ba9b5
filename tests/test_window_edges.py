"""What torch's graph and the C boundary make of window attention's calls that other
tests do not make, without a GPU."""
import pytest

torch = pytest.importorskip("torch")
from sym_amd import attention as A  # noqa: E402


class Ctx:
    device = 0


@pytest.fixture
def sums(monkeypatch):
    """window_attention as q + k + v whose lse is q's sum, and a backward that gives what it got as lse."""
    def forward(ctx, q, k, v, starts, window, sinks, scale, out, lse):
        lse.data.fill_(float(q.detach().sum()))  # by its address: torch does not count it
        return q + k + v

    def backward(ctx, dout, q, k, v, out, lse, starts, **see):
        return tuple(torch.full_like(x, float(lse[0, 0])) for x in (q, k, v))
    monkeypatch.setattr(A, "_window_attention", forward)
    monkeypatch.setattr(A, "window_attention_backward", backward)


def test_one_lse_buffer_for_two_calls(sums):
    """Each backward has the numbers of its own forward, and the buffer the last one's."""
    buffer = torch.zeros((2, 3))
    leaves = [torch.full((3, 2, 8), x).requires_grad_() for x in (1.0, 2.0)]
    outs = [A.window_attention(Ctx, q, q.detach(), q.detach(), None, window=2, lse=buffer) for q in leaves]
    assert (buffer == 96.0).all()
    for q, out in zip(leaves, outs):
        out.sum().backward()
    assert (leaves[0].grad == 48.0).all() and (leaves[1].grad == 96.0).all()
