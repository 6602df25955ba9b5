"""What torch's graph and the C boundary make of window attention's calls that other
tests do not make, without a GPU."""
import ctypes
import random

import pytest

torch = pytest.importorskip("torch")
from torch.autograd import forward_ad as F  # noqa: E402
from sym_amd import _native as N  # noqa: E402
from sym_amd import attention as A  # noqa: E402
from tests.test_window_api import refused, window_args  # noqa: E402


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


# ------------------------------------------------------------ forward mode

def calls():
    """Each call by name, with the operands that may carry a derivative."""
    h = [torch.zeros((2, n, 8), dtype=torch.float16) for n in (4, 2, 2)]
    cache = [torch.zeros((3, 16, 2, 8), dtype=torch.float16) for _ in range(2)]
    codes = [torch.zeros((3, 16, 2, 8), dtype=torch.int8) for _ in range(2)]
    scales = [torch.ones((3, 1, 2)) for _ in range(2)]
    i32 = torch.zeros(3, dtype=torch.int32)
    w, cos, sin = torch.ones(8, dtype=torch.float16), torch.ones((1, 4)), torch.ones((1, 4))
    step = i32[:2, None], i32[:2], i32
    return {
        "norm_rotate": (lambda q, k, w, c, s: A.norm_rotate(Ctx, q, k, i32[:2], c, s, w, None, 1e-6), [*h[:2], w, cos, sin]),
        "norm_rotate_backward": (lambda dq, dk, q, w: A.norm_rotate_backward(Ctx, dq, dk, q, h[1], i32[:2], cos, sin, w, None, 1e-6),
                                 [*h[:2], h[0], w]),
        "norm_rotate_append": (lambda q, k, v, w, c: A.norm_rotate_append(Ctx, q, k, v, torch.zeros(2, dtype=torch.int64), *cache,
                                                                          i32[:2], c, sin, w, None, 1e-6), [*h, w, cos]),
        "block_append": (lambda k, v: A.block_append(Ctx, k, v, *codes, *scales, *step), h[1:]),
        "tree_attention": (lambda q, k, v: A.tree_attention(Ctx, q, k, v, *step), [h[0], *cache]),
        "window_attention": (lambda q, k, v: A.window_attention(Ctx, q, k, v, i32), h),
        "window_attention_backward": (lambda d, q, k, v: A.window_attention_backward(Ctx, d, q, k, v, h[0], torch.zeros((4, 2)), i32),
                                      [h[0], *h]),
    }


@pytest.mark.parametrize("name", list(calls()))
def test_a_forward_mode_derivative_raises(monkeypatch, name):
    """It does not end in a result that says zero; without one the call runs, in such a block too."""
    made = []
    monkeypatch.setattr(A, "_call", lambda name, ctx, *args: made.append(name))
    monkeypatch.setattr(A, "_device", lambda ctx, like: like.get_device())
    monkeypatch.setattr(A, "_stream", lambda device: 0)
    monkeypatch.setattr(A, "_rotate_room", lambda *sizes: 64)
    monkeypatch.setattr(A, "_window_room", lambda *sizes: 64)
    call, operands = calls()[name]
    call(*operands)
    with F.dual_level():
        call(*operands)
        assert made == ["relx_" + name] * 2
        for i, t in enumerate(operands):
            dual = [F.make_dual(t, torch.ones_like(t)) if k == i else x for k, x in enumerate(operands)]
            for grad in (torch.enable_grad, torch.no_grad):
                with grad(), pytest.raises(RuntimeError, match="sym_amd.attention.%s has no forward-mode derivative" % name):
                    call(*dual)
        call(*operands)
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(lambda q: call(q, *operands[1:]), (operands[0],), (operands[0],))
    assert made == ["relx_" + name] * 3


def test_a_forward_mode_derivative_of_a_gradient_raises(monkeypatch):
    monkeypatch.setattr(A, "_window_attention", lambda ctx, q, k, v, starts, window, sinks, scale, out, lse: q + k + v)
    q = torch.ones((3, 2, 8)).requires_grad_()
    out = A.window_attention(Ctx, q, q.detach(), q.detach(), torch.zeros(2, dtype=torch.int32))
    with F.dual_level(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.autograd.grad(out, q, F.make_dual(torch.ones_like(out), torch.ones_like(out)))


# ------------------------------------------------------------ sizes

def workspace(**more):
    n, err = ctypes.c_size_t(), N.relx_err()
    assert N.lib().relx_window_attention_workspace(bytes(window_args(**more)), ctypes.byref(n), ctypes.byref(err)) == 0
    return n.value


@pytest.mark.parametrize("window", [0, 100, 2 ** 62])
def test_first_tokens_of_a_window_that_no_row_leaves(window):
    """However many: every row sees them without."""
    for sinks in (257, 2 ** 40):
        args = window_args(rows=100, window=window, sinks=sinks)
        assert "null context" in refused(N.lib().relx_window_attention, None, bytes(args), 0)[1]
        assert workspace(rows=100, window=window, sinks=sinks) == workspace(rows=100, window=0, sinks=0)
    if window:
        more = window_args(rows=101, window=min(window, 100), sinks=257)
        assert refused(N.lib().relx_window_attention, None, bytes(more), 0)[0] == "unsupported_layout"


def test_a_workspace_of_short_sequences():
    """First tokens' sums are of sequences that some window leaves: 4096 of 32 rows, within a
    window of 1024, have room for as many as could be longer, and not for all of them."""
    a_piece = 8 * 256 * 2 * 128 * 4
    stats = 32 * 2 ** 17 * 2 * 4
    sizes = dict(rows=2 ** 17, heads=32, kv_heads=8, dim=128, sinks=256, window=1024)
    assert workspace(sequences=4096, **sizes) <= stats + (2 ** 17 // 4096 + 2 ** 17 // 1025 + 2) * a_piece
    assert workspace(sequences=5, **sizes) == stats + (2 ** 17 // 4096 + 5 + 2) * a_piece  # all of a few

    # the numbers of pieces: each of its own, in order, and within the room
    rng = random.Random(1)
    for _ in range(300):
        window, size = rng.randint(1, 60), rng.choice([32, 96, 128])
        lengths = [rng.choice([0, 1, window, window + 1, rng.randint(0, 400)]) for _ in range(rng.randint(0, 40))]
        before, after = rng.randint(0, 90), rng.randint(0, 90)
        rows, at, taken = before + sum(lengths) + after, before, -1
        for b, n in enumerate(lengths, 1):
            first = at // size + min(b, at // (window + 1))
            if n > window:
                assert first > taken
                taken = first + -(-n // size) - 1
            at += n
            if b < len(lengths):  # the next sequence's is beyond: a search for the last that is not ends here
                assert at // size + min(b + 1, at // (window + 1)) > taken
        assert taken < rows // size + min(len(lengths), rows // (window + 1)) + 2


def test_no_window_is_none_or_zero():
    assert A._reach(None, 0) == A._reach(0, 0) == (0, 0) and A._reach(10 ** 30, 3) == (2 ** 62, 3)
    for window in (None, 0):
        with pytest.raises(ValueError, match="first ones"):
            A._reach(window, 2)


def test_gradients_are_laid_out_for_the_kernels():
    """As they lie where the kernels take them so, else as a copy of the same numbers."""
    x = torch.randn((5, 4, 16)).half()
    room = torch.zeros(x.numel() + 1, dtype=torch.float16)
    room[1:] = x.flatten()
    wide = torch.zeros((5, 4, 20), dtype=torch.float16)
    wide[..., :16] = x
    far = torch.empty_strided((1, 4, 16), ((1 << 24) + 8, 16, 1), dtype=torch.float16).copy_(x[:1])
    assert A._packed(x) is x and A._packed(x[:, 1:3]).data_ptr() == x[:, 1:3].data_ptr()
    one = torch.tensor(2.0, dtype=torch.float16).expand(5, 4, 16)
    for t in (room[1:].view(5, 4, 16), room.new_zeros(x.numel() + 3)[3:].view(5, 4, 16), wide[..., :16], one, x[:1].expand(5, 4, 16),
              x.transpose(1, 2).contiguous().transpose(1, 2), far):
        p = A._packed(t)
        assert torch.equal(p, t) and p.is_contiguous() and p.data_ptr() % 16 == 0 and p.data_ptr() != t.data_ptr()
