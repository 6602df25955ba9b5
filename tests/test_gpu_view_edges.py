"""What reaches a result of attention over a cache with a window, and what must not:
scales of blocks that a row does not see, bits of a mask beyond a request's rows, tokens
beyond a table."""
import pytest

from tests import window_cases as W
from tests.test_gpu_blocks import check_view, on_gpu

torch = pytest.importorskip("torch")
from sym_amd import attention as A  # noqa: E402
from sym_amd import pyreloc as P  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, I8 = torch.float16, torch.bfloat16, torch.int8
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def ctx():
    c = P.Context(0)
    yield c
    c.close()


# ------------------------------------------------------------ scales of blocks

def seen_blocks(s, window, sinks):
    """[rows, pages, page / block]: whether a row sees a token of the block."""
    pages, page = s["cache_k"].shape[:2]
    blocks = s["k_scale"].shape[1]
    out = torch.zeros((s["q"].shape[0], pages, blocks), dtype=torch.bool)
    for b in range(s["table"].shape[0]):
        r0, r1, c = int(s["starts"][b]), int(s["starts"][b + 1]), int(s["cached"][b])
        for j in range(r1 - r0):
            words = None if s["mask"] is None else [w & (2 ** 64 - 1) for w in s["mask"][r0 + j].tolist()]
            depth = j if words is None else sum(bin(w).count("1") for w in words) - 1
            for x in range(min(c + r1 - r0, s["table"].shape[1] * page)):
                new = x - c
                own = new < 0 or (new <= j if words is None else words[new // 64] >> (new % 64) & 1)
                near = x < sinks or c + depth - x < window or (words is not None and new >= 0)
                if own and near:
                    out[r0 + j, int(s["table"][b, x // page]), x % page * blocks // page] = True
    return out


def attend(ctx, s, window, sinks):
    d = on_gpu(s)
    return A.tree_attention(ctx, d["q"], d["cache_k"], d["cache_v"], d["table"], d["cached"], d["starts"], mask=d["mask"],
                            scale=d["scale"], k_scale=d["k_scale"], v_scale=d["v_scale"], window=window, sinks=sinks).cpu()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("cached,fresh,heads,kv,dim,page,window,sinks,columns", [
    ([460], [2], 4, 2, 64, 16, 89, 4, 32),               # a table that is not cut
    ([600], [1], 4, 2, 128, 16, 101, 4, None),
    ([600, 77], [2, 1], 4, 2, 64, 48, 101, 40, None),
    ([600], [1], 8, 4, 128, 16, 101, 4, 2048),           # four heads at a time
    ([600], [40], 4, 2, 128, 16, 101, 4, None),          # more rows than 16
    ([600, 200], [40, 30], 4, 2, 64, 48, 101, 20, None),
    ([600], [30], 2, 2, 256, 16, 101, 4, None),
    ([600], [1], 4, 2, 72, 16, 101, 4, None),            # through registers
    ([600], [40], 4, 2, 72, 16, 101, 4, None),
])
def test_scales_that_no_row_sees(ctx, dtype, cached, fresh, heads, kv, dim, page, window, sinks, columns):
    """A half of a tile that lies before every row's window, behind the first tokens or
    behind the last: its scales may be anything, and leave every bit as it is."""
    s = W.view_case(21, cached, fresh, heads, kv, dim, dtype, I8, page, 16, columns=columns)
    begin = cached[0] - window + 1  # of the first row's window
    assert begin % 32 >= 16
    want = check_view(ctx, s, "scales %s" % [cached, fresh, dim, page], window, sinks).cpu()
    nobody = ~seen_blocks(s, window, sinks).any(0)
    half = begin - begin % 16 - 1  # the last token of the tile's other half
    assert nobody[int(s["table"][0, half // page]), half % page // 16]
    for bad in (INF, NAN, 1e30, 3e38):
        t = dict(s, k_scale=s["k_scale"].clone(), v_scale=s["v_scale"].clone())
        t["k_scale"][nobody] = bad
        t["v_scale"][nobody] = bad
        assert torch.equal(attend(ctx, t, window, sinks), want), bad


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("fresh,words", [(12, 0), (40, 0), (9, 1), (50, 1), (100, 2)])
def test_scales_that_other_rows_see(ctx, dtype, fresh, words):
    """Of a block that some rows of an item see: nothing of it in the others."""
    window, sinks = (24, 2) if not words else (128, 2)
    s = W.view_case(22, [300], [fresh], 2, 1, 64, dtype, I8, 16, 16, tree_words=words)
    want = check_view(ctx, s, "rows %s" % [fresh, words], window, sinks).cpu()
    sees = seen_blocks(s, window, sinks)
    some = (sees.any(0) & ~sees.all(0)).nonzero().tolist()
    assert some
    for at in some:
        rows = sees[:, at[0], at[1]]
        for bad in (INF, 3e38):
            t = dict(s, v_scale=s["v_scale"].clone())
            t["v_scale"][at[0], at[1]] = bad
            assert torch.equal(attend(ctx, t, window, sinks)[~rows], want[~rows]), (at, bad)


# ------------------------------------------------------------ masks

@pytest.mark.parametrize("cache", ["own", "blocks"])
@pytest.mark.parametrize("fresh,words", [([1, 5, 2], 1), ([3, 70, 1], 2)])
def test_bits_beyond_a_requests_rows(ctx, cache, fresh, words):
    """A mask's bits of tokens that a request does not add say nothing, of depths neither."""
    window = 64 * words
    s = W.view_case(23, [500, 90, 333], fresh, 4, 2, 64, BF16, BF16 if cache == "own" else I8, 32, 16 if cache == "blocks" else None,
                    tree_words=words)
    want = check_view(ctx, s, "bits %s" % fresh, window, 3).cpu()
    mask = s["mask"].clone()
    for b, n in enumerate(fresh):
        for w in range(words):
            beyond = (2 ** 64 - 1) ^ (2 ** min(max(n - 64 * w, 0), 64) - 1)
            mask[int(s["starts"][b]):int(s["starts"][b + 1]), w] |= beyond - (2 ** 64 if beyond >> 63 else 0)
    assert not torch.equal(mask, s["mask"])
    assert torch.equal(attend(ctx, dict(s, mask=mask), window, 3), want)


# ------------------------------------------------------------ tables

@pytest.mark.parametrize("cache", ["own", "int8", "blocks"])
@pytest.mark.parametrize("cached,fresh,dim,page,columns,window,sinks,words", [
    ([63, 5], [2, 1], 64, 32, 1, 20, 1, 0),
    ([700, 40], [1, 1], 128, 64, 9, 300, 33, 0),
    ([700, 640], [40, 9], 64, 64, 10, 130, 3, 0),
    ([500, 90], [3, 30], 64, 32, 7, 300, 0, 2),
    ([500], [1], 64, 16, 10, 100, 0, 0),  # nothing of the window is left
])
def test_a_table_that_holds_fewer_than_the_cached_tokens(ctx, cache, cached, fresh, dim, page, columns, window, sinks, words):
    """Positions go by the cached tokens, those in the table or not."""
    for dtype in (F16, BF16):
        s = W.view_case(24, cached, fresh, 4, 2, dim, dtype, dtype if cache == "own" else I8, page, 16 if cache == "blocks" else None,
                        tree_words=words, columns=columns)
        check_view(ctx, s, "short table %s" % [cached, columns], window, sinks)
