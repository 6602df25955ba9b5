"""Tree attention over contexts so long that every wave reads many tiles, at each
of its forms: tiles go round their rings, table entries come in many batches and
a row's sum has many parts. Few pages are listed over and over, so the
definition in 64 bits needs only how often each slot is seen."""
import random

import pytest

from tests import attention_cases as C

torch = pytest.importorskip("torch")
from sym_amd import attention as A  # noqa: E402
from sym_amd import pyreloc as P  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, I8 = torch.float16, torch.bfloat16, torch.int8


@pytest.fixture(scope="module")
def ctx():
    c = P.Context(0)
    yield c
    c.close()


def definition(q, keys, values, table, cached, mask, scale, round_to):
    """(result, log of sums, bound of the result) of one request."""
    pages, page, kv, dim = keys.shape
    fresh, heads, _ = q.shape
    at = table.long().repeat_interleave(page) * page + torch.arange(table.numel() * page) % page
    often = torch.bincount(at[:cached], minlength=pages * page).double()
    n = torch.zeros((fresh, pages * page), dtype=torch.float64)
    for j in range(fresh):
        n[j] = often + torch.bincount(at[cached:cached + fresh][mask[j]], minlength=pages * page)
    group, u = heads // kv, C.ROUND[round_to]
    k, v = (x.double().reshape(pages * page, kv, dim).repeat_interleave(group, 1) for x in (keys, values))
    s = torch.stack([q[:, h].double() @ k[:, h].T for h in range(heads)], 1) * scale  # [fresh, heads, slots]
    s = s + n.log()[:, None]
    lse = torch.logsumexp(s, 2)
    p = (s - lse[..., None]).exp()
    out = torch.stack([p[:, h] @ v[:, h] for h in range(heads)], 1)
    size = torch.stack([p[:, h] @ v[:, h].abs() for h in range(heads)], 1)
    ds = (dim + 4) * C.F32 * float((k.abs().amax((0, 1)) * q.double().abs().amax((0, 1))).sum()) * scale
    steps = (cached + fresh) / 32 + 16
    bound = u * out.abs() + (u + 2 * ds + steps * C.F32) * size + (cached + fresh) * 2.0 ** -31 * v.abs().max() + 2.0 ** -24
    return out, lse, bound


# rows that share a key head: up to 16, 64, 128, 256; a mask of one word, of two
@pytest.mark.parametrize("heads,kv,fresh,dim", [(32, 32, 1, 64), (32, 32, 3, 128), (16, 8, 13, 128), (16, 8, 50, 128),
                                                (16, 8, 100, 128), (16, 8, 100, 64), (6, 6, 40, 200), (32, 32, 2, 256)])
@pytest.mark.parametrize("page,dtype,cache", [(16, BF16, BF16), (32, F16, F16), (24, F16, F16), (16, F16, I8), (40, BF16, I8)])
def test_tree_attention_over_many_tiles_a_wave(ctx, heads, kv, fresh, dim, page, dtype, cache):
    print("[gpu-case] long", heads, kv, fresh, dim, page, dtype, cache, flush=True)
    gen = torch.Generator().manual_seed(heads + fresh + dim + page)
    cached, pages = 150_003, 24
    columns = -(-(cached + fresh) // page)
    table = torch.randint(0, pages, (columns,), generator=gen, dtype=torch.int32)
    made, scales = [], [None, None]
    for i in range(2):
        if cache == I8:
            made.append(torch.randint(-127, 128, (pages, page, kv, dim), generator=gen, dtype=I8))
            scales[i] = torch.rand(kv, generator=gen) * 0.01 + 0.005
        else:
            made.append(torch.randn((pages, page, kv, dim), generator=gen).to(cache))
    q = torch.randn((fresh, heads, dim), generator=gen).to(dtype)
    words = -(-fresh // 64)
    bits = C.tree_mask(C.tree(random.Random(fresh), fresh), words)
    mask = torch.tensor([[r[j >> 6] >> (j & 63) & 1 for j in range(fresh)] for r in bits], dtype=torch.bool)
    lse = torch.empty((fresh, heads), device=DEV)
    out = A.tree_attention(ctx, q.to(DEV), made[0].to(DEV), made[1].to(DEV), table[None].to(DEV),
                           torch.tensor([cached], dtype=torch.int32, device=DEV),
                           torch.tensor([0, fresh], dtype=torch.int32, device=DEV),
                           mask=torch.tensor(bits, dtype=torch.int64, device=DEV), lse=lse,
                           **({} if cache != I8 else dict(k_scale=scales[0].to(DEV), v_scale=scales[1].to(DEV))))
    torch.cuda.synchronize()
    k, v = (m if c is None else m.double() * c.double()[:, None] for m, c in zip(made, scales))
    want, want_lse, bound = definition(q, k, v, table, cached, mask, dim ** -0.5, dtype)
    assert bool(((out.double().cpu() - want).abs() <= bound).all())
    # a tile left out would be 32 tokens in 150000: twice this
    assert bool(((lse.double().cpu() - want_lse).abs() <= 2.0 ** -17 * (1 + want_lse.abs())).all())
