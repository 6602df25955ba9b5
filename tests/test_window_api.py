"""The boundary of window attention and of caches with a scale a block, without a
GPU: records, refusals before a device is looked at, the gradients' formula, and
what torch's graph sees."""
import ctypes
import os
import random
import re

import pytest

from tests import window_cases as W

torch = pytest.importorskip("torch")
from sym_amd import _native as N  # noqa: E402
from sym_amd import attention as A  # noqa: E402

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "relx.h")
ADDRESS = 1 << 20  # never followed


@pytest.fixture(scope="module")
def lib():
    return N.lib()


def refused(fn, *args):
    err = N.relx_err()
    assert fn(*args, ctypes.byref(err)) != 0
    return err.code.decode(), err.message.decode()


@pytest.mark.parametrize("name", ["relx_block_scales", "relx_cache_view", "relx_block_append_args", "relx_window_args"])
def test_records_are_the_headers(name):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), open(HEADER).read(), re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = [re.sub(r"\W", "", part.split()[-1]) for line in body.split(";") if line.strip() for part in line.split(",")]
    record = getattr(N, name)
    assert [f for f, _ in record._fields_] == fields
    assert ctypes.sizeof(record) == 8 * len(A._format(record))


# ------------------------------------------------------------ packed sequences

def window_args(**more):
    a = N.relx_window_args()
    d = dict(rows=100, sequences=2, heads=8, kv_heads=2, dim=64, window=16, sinks=2, kind=1, bits=16, scale=0.125,
             starts=ADDRESS, lse=ADDRESS)
    d.update(more)
    for k, v in d.items():
        if k not in ("q", "k", "v", "out"):
            setattr(a, k, v)
    for n, h in (("q", a.heads), ("k", a.kv_heads), ("v", a.kv_heads), ("out", a.heads)):
        data, row, head = more.get(n, (ADDRESS, h * a.dim, a.dim))
        r = getattr(a, n)
        r.data, r.row, r.head = data, row, head
    return a


BAD_WINDOWS = [
    ("invalid_argument", dict(rows=-1)), ("invalid_argument", dict(rows=2 ** 31)), ("invalid_argument", dict(sequences=-1)),
    ("invalid_argument", dict(kv_heads=3)), ("invalid_argument", dict(kv_heads=0)), ("invalid_argument", dict(heads=0)),
    ("invalid_argument", dict(window=-1)), ("invalid_argument", dict(sinks=-1)), ("invalid_argument", dict(scale=float("inf"))),
    ("invalid_argument", dict(scale=float("nan"))), ("invalid_argument", dict(starts=None)),
    ("unsupported_layout", dict(rows=2 ** 29 + 1, heads=1, kv_heads=1)), ("unsupported_layout", dict(dim=136)), ("unsupported_layout", dict(dim=4)),
    ("unsupported_layout", dict(dim=60)), ("unsupported_layout", dict(sinks=257)), ("unsupported_layout", dict(kind=0, bits=32)),
    ("unsupported_layout", dict(kind=2, bits=8)), ("unsupported_layout", dict(kind=7)),
    ("unsupported_layout", dict(heads=65536, kv_heads=1)), ("unsupported_layout", dict(rows=2 ** 28, heads=32, kv_heads=32)),
    ("unsupported_layout", dict(sequences=2 ** 24)),
]


@pytest.mark.parametrize("code,bad", BAD_WINDOWS)
def test_window_attention_refuses_sizes(lib, code, bad):
    args = bytes(window_args(**bad))
    assert refused(lib.relx_window_attention, None, args, 0)[0] == code
    assert refused(lib.relx_window_attention_backward, None, args, None, None, None, None, None, 0, 0)[0] == code
    if bad != dict(starts=None):  # sizes alone count there
        assert refused(lib.relx_window_attention_workspace, args, ctypes.byref(ctypes.c_size_t()))[0] == code


@pytest.mark.parametrize("code,bad", [
    ("invalid_argument", dict(q=(None, 512, 64))), ("invalid_argument", dict(out=(None, 512, 64))),
    ("invalid_argument", dict(k=(ADDRESS, -128, 64))), ("invalid_argument", dict(out=(ADDRESS, 0, 64))),
    ("invalid_argument", dict(out=(ADDRESS, 512, 32))), ("unsupported_layout", dict(q=(ADDRESS + 2, 512, 64))),
    ("unsupported_layout", dict(v=(ADDRESS, 130, 64))), ("unsupported_layout", dict(k=(ADDRESS, 128, 4))),
    ("unsupported_layout", dict(q=(ADDRESS, 2 ** 24 + 8, 64))),
])
def test_window_attention_refuses_layouts(lib, code, bad):
    assert refused(lib.relx_window_attention, None, bytes(window_args(**bad)), 0)[0] == code


def test_window_attention_takes_the_rest(lib):
    """Refused for the want of a context alone."""
    for good in (dict(), dict(window=0, sinks=0), dict(sinks=256), dict(window=2 ** 62), dict(lse=None), dict(dim=8), dict(dim=128),
                 dict(rows=0, starts=None), dict(sequences=0), dict(heads=40, kv_heads=1), dict(scale=0.0), dict(scale=-1.0),
                 dict(rows=1, q=(ADDRESS, 3, 64)), dict(k=(ADDRESS, 0, 64), v=(ADDRESS, 64, 0))):
        assert "null context" in refused(lib.relx_window_attention, None, bytes(window_args(**good)), 0)[1], good


def test_the_backward_takes_a_workspace_and_lse(lib):
    def back(args, room, size, **more):
        heads = {n: N.relx_heads(*more.get(n, (ADDRESS, h * 64, 64))) for n, h in (("do", 8), ("dq", 8), ("dk", 2), ("dv", 2))}
        return refused(lib.relx_window_attention_backward, None, bytes(args), *(bytes(heads[n]) for n in ("do", "dq", "dk", "dv")),
                       room, size, 0)
    size = ctypes.c_size_t()
    err = N.relx_err()
    args = window_args()
    assert lib.relx_window_attention_workspace(bytes(args), ctypes.byref(size), ctypes.byref(err)) == 0
    assert size.value >= 2 * 8 * 100 * 4
    assert "null context" in back(args, ADDRESS, size.value)[1]
    assert back(args, ADDRESS, size.value - 1)[0] == "insufficient_capacity"
    assert back(args, None, size.value)[0] == "insufficient_capacity"
    assert back(args, ADDRESS + 4, size.value)[0] == "invalid_argument"
    assert back(window_args(lse=None), ADDRESS, size.value)[0] == "invalid_argument"
    for name in ("dq", "dk", "dv"):
        assert back(args, ADDRESS, size.value, **{name: (ADDRESS, 0, 64)})[0] == "invalid_argument"
        assert back(args, ADDRESS, size.value, **{name: (None, 512, 64)})[0] == "invalid_argument"


def test_workspaces_grow_with_what_they_hold(lib):
    def size(**more):
        n, err = ctypes.c_size_t(), N.relx_err()
        assert lib.relx_window_attention_workspace(bytes(window_args(**more)), ctypes.byref(n), ctypes.byref(err)) == 0
        return n.value
    assert size(rows=0) < size() < size(rows=1000) < size(rows=1000, sinks=256)
    assert size(rows=1000, sinks=256, window=1000) == size(rows=1000, sinks=0)  # no row leaves the window
    assert size(rows=2 ** 20, heads=32, kv_heads=8, sinks=4, window=1024, dim=128) < 1 << 30


# ------------------------------------------------------------ blocks of a cache

def append_args(**more):
    a = N.relx_block_append_args()
    d = dict(rows=10, requests=2, columns=4, kind=1, bits=16, table=ADDRESS, table_row=4, cached=ADDRESS, starts=ADDRESS)
    c = dict(keys=ADDRESS, values=ADDRESS, key_page=32 * 2 * 64, key_slot=2 * 64, key_head=64, value_page=32 * 2 * 64,
             value_slot=2 * 64, value_head=64, pages=8, page=32, kv_heads=2, dim=64, kind=2, bits=8)
    s = dict(key_scale=ADDRESS, value_scale=ADDRESS, page=4, block_stride=2, head=1, block=16)
    for target, fields, prefix in ((a, d, ""), (a.cache, c, "cache_"), (a.scales, s, "scale_")):
        for k, v in fields.items():
            setattr(target, k, more.pop(prefix + k, v))
    for n in ("k", "v"):
        h = getattr(a, n)
        h.data, h.row, h.head = more.pop(n, (ADDRESS, 128, 64))
    assert not more, more
    return a


@pytest.mark.parametrize("code,bad", [
    ("invalid_argument", dict(rows=-1)), ("invalid_argument", dict(requests=2 ** 31)), ("invalid_argument", dict(columns=-1)),
    ("invalid_argument", dict(table=None)), ("invalid_argument", dict(cached=None)), ("invalid_argument", dict(starts=None)),
    ("invalid_argument", dict(k=(None, 128, 64))), ("invalid_argument", dict(cache_keys=None)),
    ("invalid_argument", dict(scale_value_scale=None)), ("invalid_argument", dict(scale_page=-1)),
    ("invalid_argument", dict(scale_page=2)), ("invalid_argument", dict(scale_head=0)),
    ("invalid_argument", dict(cache_key_page=64)), ("invalid_argument", dict(cache_value_head=32)),
    ("invalid_argument", dict(cache_key_slot=-64)), ("invalid_argument", dict(cache_page=0)),
    ("unsupported_layout", dict(kind=2, bits=8)), ("unsupported_layout", dict(cache_kind=1, cache_bits=16)),
    ("unsupported_layout", dict(scale_block=8)), ("unsupported_layout", dict(scale_block=24)),
    ("unsupported_layout", dict(scale_block=64)), ("unsupported_layout", dict(scale_block=0)),
    ("unsupported_layout", dict(cache_dim=513)), ("unsupported_layout", dict(columns=2 ** 26)),
    ("unsupported_layout", dict(rows=2 ** 29)), ("unsupported_layout", dict(requests=2 ** 23)),
])
def test_block_append_refuses(lib, code, bad):
    assert refused(lib.relx_block_append, None, bytes(append_args(**bad)), 0)[0] == code


def test_block_append_takes_the_rest(lib):
    for good in (dict(), dict(kind=0, bits=32), dict(kind=0, bits=16), dict(cache_dim=7, cache_kv_heads=1), dict(rows=0, k=(None, 0, 0)),
                 dict(requests=0, table=None), dict(scale_block=32, scale_block_stride=0), dict(k=(ADDRESS + 2, 129, 64)),
                 dict(cache_pages=0, cache_keys=None)):
        assert "null context" in refused(lib.relx_block_append, None, bytes(append_args(**good)), 0)[1], good


def test_a_view_refuses(lib):
    def go(view, **more):
        a = N.relx_tree_attention_args()
        for k, v in dict(dict(rows=0, requests=1, heads=4, columns=2, kind=1, bits=16, cached=ADDRESS, starts=ADDRESS,
                              table=ADDRESS, words=0), **more).items():
            setattr(a, k, v)
        for k, v in dict(keys=ADDRESS, values=ADDRESS, pages=4, page=32, kv_heads=2, dim=64, kind=2, bits=8, key_scale=ADDRESS,
                         value_scale=ADDRESS).items():
            setattr(a.cache, k, v)
        w = N.relx_cache_view()
        for k, v in view.items():
            setattr(w if hasattr(w, k) else w.scales, k, v)
        return refused(lib.relx_tree_attention_view, None, bytes(a), bytes(w), 0)
    blocks = dict(key_scale=ADDRESS, value_scale=ADDRESS, block=16, page=4, block_stride=2, head=1)
    assert "null context" in go({})[1] and "null context" in go(blocks)[1] and "null context" in go(dict(window=5, sinks=1))[1]
    assert "null context" in go(dict(window=128), mask=ADDRESS, words=2)[1]
    assert go(dict(window=127), mask=ADDRESS, words=2)[0] == "unsupported_layout"
    assert go(dict(window=-1))[0] == go(dict(sinks=-1))[0] == "invalid_argument"
    assert go(dict(blocks, block=8))[0] == go(dict(blocks, block=48))[0] == "unsupported_layout"
    assert go(dict(blocks, value_scale=None))[0] == go(dict(blocks, head=-1))[0] == "invalid_argument"
    assert go(dict(blocks, page=2 ** 29))[0] == "unsupported_layout"  # further apart than a lane's distance holds
    assert refused(lib.relx_tree_attention_view, None, bytes(N.relx_tree_attention_args()), None, 0)[0] == "invalid_argument"


# ------------------------------------------------------------ formulas

@pytest.mark.parametrize("window,sinks", [(None, 0), (3, 0), (2, 2)])
def test_the_gradients_formula_against_differences(window, sinks):
    s = {k: v.double() if v.is_floating_point() else v for k, v in W.window_case(1, [7, 4], 4, 2, 8, torch.float16).items()}

    def value(q, k, v):
        out = W.window_attention(q, k, v, s["starts"], window, sinks, 0.4, round_to=torch.float16)
        return float((out["o"] * s["dout"]).sum())
    want = W.window_attention(s["q"], s["k"], s["v"], s["starts"], window, sinks, 0.4, s["dout"], torch.float16)
    rng, h = random.Random(1), 1e-5
    for at, name in enumerate(("dq", "dk", "dv")):
        for _ in range(12):
            i = tuple(rng.randrange(n) for n in want[name].shape)
            ends = []
            for sign in (1, -1):
                moved = [s[n].clone() for n in "qkv"]
                moved[at][i] += sign * h
                ends.append(value(*moved))
            assert abs((ends[0] - ends[1]) / (2 * h) - float(want[name][i])) < 1e-7


def test_a_blocks_codes_by_hand():
    """Two tokens, then a larger one: the first two are rounded anew."""
    cache, scale = torch.zeros((2, 16, 1, 2), dtype=torch.int8), torch.full((2, 1, 1), 9.0)
    table = torch.tensor([[1]], dtype=torch.int32)
    first = torch.tensor([[[1.27, -0.5]], [[0.004, 0.02]]])
    ck, _, ks, _ = W.block_append(first, first, cache, cache, scale, scale, table, torch.tensor([0]), torch.tensor([0, 2]))
    assert ck[1, :2, 0].tolist() == [[127, -50], [0, 2]] and abs(float(ks[1, 0, 0]) - 0.01) < 1e-8 and float(ks[0, 0, 0]) == 9.0
    more = torch.tensor([[[2.54, 0.0]]])
    ck, _, ks, _ = W.block_append(more, more, ck, ck, ks, ks, table, torch.tensor([2]), torch.tensor([0, 1]))
    assert ck[1, :3, 0].tolist() == [[64, -25], [0, 1], [127, 0]] and abs(float(ks[1, 0, 0]) - 0.02) < 1e-8


# ------------------------------------------------------------ torch's graph

class Ctx:
    device = 0


def test_derivatives(monkeypatch):
    """Of window_attention as q + k + v, once, and only where they are wanted."""
    seen = []

    def forward(ctx, q, k, v, starts, window, sinks, scale, out, lse):
        assert lse is not None
        return q + k + v

    def backward(ctx, dout, q, k, v, out, lse, starts, **see):
        seen.append(see)
        return dout, 2 * dout, 3 * dout
    monkeypatch.setattr(A, "_window_attention", forward)
    monkeypatch.setattr(A, "window_attention_backward", backward)
    q, k, v = (torch.ones((3, 2, 8)).requires_grad_(n != "k") for n in "qkv")
    o = A.window_attention(Ctx, q, k, v, torch.tensor([0, 3]), window=2, sinks=1, scale=0.5)
    o.sum().backward()
    assert torch.equal(q.grad, torch.ones_like(q)) and k.grad is None and torch.equal(v.grad, 3 * torch.ones_like(v))
    assert seen == [dict(window=2, sinks=1, scale=0.5)]
    g, = torch.autograd.grad((A.window_attention(Ctx, q, k, v, None, window=2) ** 2).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (g ** 2).sum().backward()


def test_calls_without_a_gradient_say_so(monkeypatch):
    monkeypatch.setattr(A, "_call", lambda name, ctx, *args: None)
    monkeypatch.setattr(A, "_device", lambda ctx, like: like.get_device())
    monkeypatch.setattr(A, "_stream", lambda device: 0)
    i32 = torch.zeros(3, dtype=torch.int32)
    q = torch.zeros((2, 4, 8), dtype=torch.float16).requires_grad_()
    cache = torch.zeros((3, 32, 2, 8), dtype=torch.int8)
    scale = torch.ones((3, 2, 2))
    out = A.tree_attention(Ctx, q, cache, cache, i32[:2, None], i32[:2], i32, k_scale=scale, v_scale=scale, window=9, sinks=1)
    with pytest.raises(RuntimeError, match="no gradient"):
        out.float().sum().backward()
    k = torch.zeros((2, 2, 8), dtype=torch.float16).requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        A.block_append(Ctx, k, k.detach(), cache, cache, scale, scale, i32[:2, None], i32[:2], i32)
    with torch.no_grad():
        A.block_append(Ctx, k, k, cache, cache, scale, scale, i32[:2, None], i32[:2], i32)
