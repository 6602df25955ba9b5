"""What torch's graph sees of the paged-cache operators, on the CPU: the calls of
the library are replaced by functions of the same shape."""
import pytest

torch = pytest.importorskip("torch")
from sym_amd import attention as A  # noqa: E402


class Ctx:
    device = 0


@pytest.fixture
def squares(monkeypatch):
    """norm_rotate as q^2 w and k^2 w, and its gradients."""
    def forward(ctx, q, k, positions, cos, sin, qw, kw, eps, pairs, out):
        return q * q * (1 if qw is None else qw), k * k * (1 if kw is None else kw)

    def backward(ctx, dq, dk, q, k, positions, cos, sin, qw, kw, eps, pairs=False, **more):
        grads = [2 * x * d * (1 if w is None else w) for x, d, w in ((q, dq, qw), (k, dk, kw))]
        return (*grads, *(None if w is None else (x * x * d).sum((0, 1)) for x, d, w in ((q, dq, qw), (k, dk, kw))))
    monkeypatch.setattr(A, "_norm_rotate", forward)
    monkeypatch.setattr(A, "norm_rotate_backward", backward)
    gen = torch.Generator().manual_seed(1)
    q, k = (torch.randn((3, 2, 4), generator=gen).requires_grad_() for _ in range(2))
    return q, k, torch.ones((5, 2)), torch.ones((5, 2)), torch.ones(4).requires_grad_()


def test_first_derivatives(squares):
    q, k, cos, sin, w = squares
    zq, zk = A.norm_rotate(Ctx, q, k, None, cos, sin, w, None, 1e-6)
    (zq.sum() + 3 * zk.sum()).backward()
    assert torch.allclose(q.grad, 2 * q) and torch.allclose(k.grad, 6 * k) and torch.allclose(w.grad, (q * q).sum((0, 1)))
    with torch.no_grad():
        assert not A.norm_rotate(Ctx, q, k, None, cos, sin, w, None, 1e-6)[0].requires_grad


def test_a_second_derivative_raises(squares):
    q, k, cos, sin, w = squares
    zq, zk = A.norm_rotate(Ctx, q, k, None, cos, sin, w, w, 1e-6)
    grad, = torch.autograd.grad((zq ** 2).sum() + zk.sum(), q, create_graph=True)
    loss = (q ** 2).sum() + (grad ** 2).sum()  # a penalty beside another term
    with pytest.raises(RuntimeError, match="once_differentiable"):
        loss.backward()


@pytest.mark.parametrize("which", [0, 1])
def test_a_derivative_by_the_angles_raises(squares, which):
    q, k, cos, sin, _ = squares
    angles = [cos, sin]
    angles[which].requires_grad_()
    zq, _ = A.norm_rotate(Ctx, q.detach(), k.detach(), None, *angles, None, None, 1e-6)
    with pytest.raises(RuntimeError, match="cos and sin"):
        zq.sum().backward()


def test_calls_without_a_gradient_say_so(monkeypatch):
    """The result is marked, whichever operand asks; the call itself runs once, and no mark without a graph."""
    calls = []
    monkeypatch.setattr(A, "_call", lambda name, ctx, *args: calls.append(name))
    monkeypatch.setattr(A, "_device", lambda ctx, like: like.get_device())
    monkeypatch.setattr(A, "_stream", lambda device: 0)
    h = [torch.zeros((2, n, 8), dtype=torch.float16) for n in (4, 2, 2)]
    cache = [torch.zeros((3, 16, 2, 8), dtype=torch.float16) for _ in range(2)]
    i32 = torch.zeros(3, dtype=torch.int32)
    w = torch.ones(8, dtype=torch.float16)
    turn = (i32[:2], torch.ones((1, 4)), torch.ones((1, 4)), w, None, 1e-6)

    def append(**more):
        return A.norm_rotate_append(Ctx, *h, torch.zeros(2, dtype=torch.int64), *cache, *turn, **more)

    def attend(**more):
        return A.tree_attention(Ctx, h[0], *cache, i32[:, None][:2], i32[:2], i32, **more)

    for name, call, wanted in (("norm_rotate_append", append, (*h, w, turn[1])), ("tree_attention", attend, (h[0], *cache))):
        assert not call().requires_grad
        for t in wanted:
            t.requires_grad_()
            calls.clear()
            out = call()
            assert len(calls) == 1 and out.requires_grad and out.shape == h[0].shape
            with pytest.raises(RuntimeError, match="%s has no gradient" % name):
                out.float().sum().backward()
            with torch.no_grad():
                assert not call().requires_grad
            given = torch.empty_like(h[0], requires_grad=False)
            assert call(out=given) is given and not given.requires_grad
            t.requires_grad_(False)


@pytest.mark.parametrize("wanted", [(True, False), (False, True), (False, False), (True, True)])
def test_gradients_of_frozen_weights_are_not_computed(squares, monkeypatch, wanted):
    q, k, cos, sin, _ = squares
    asked = []

    def backward(ctx, dq, dk, *rest, weight_grads, **more):
        asked.append(tuple(weight_grads))
        return dq, dk, *(torch.ones(4) if w else None for w in weight_grads)
    monkeypatch.setattr(A, "norm_rotate_backward", backward)
    weights = [torch.ones(4).requires_grad_(w) for w in wanted]
    zq, zk = A.norm_rotate(Ctx, q, k, None, cos, sin, *weights, 1e-6)
    (zq.sum() + zk.sum()).backward()
    assert asked == [wanted] and [w.grad is not None for w in weights] == list(wanted)
