"""Calls of the paged-cache operators at the edges of what they take, against
their definitions (tests/attention_cases.py)."""
import pytest

from tests import attention_cases as C

torch = pytest.importorskip("torch")
from sym_amd import attention as A  # noqa: E402
from sym_amd import pyreloc as P  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32, I8 = torch.float16, torch.bfloat16, torch.float32, torch.int8


def say(*a):
    print("[gpu-case]", *a, flush=True)


@pytest.fixture(scope="module")
def ctx():
    assert torch.cuda.is_available(), "a GPU test needs the MI355X"
    c = P.Context(0)
    yield c
    c.close()


def on_gpu(s):
    return {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in s.items()}


# ------------------------------------------------------------ no requests

@pytest.mark.parametrize("dtype,cache,heads,dim,rows", [(F16, F16, 4, 64, 1), (BF16, I8, 8, 128, 9), (BF16, BF16, 6, 200, 300)])
def test_rows_without_any_request_are_zero(ctx, dtype, cache, heads, dim, rows):
    say("no requests", dtype, cache, heads, dim, rows)
    s = on_gpu(C.attention_case(1, [20], [rows], heads, 2, dim, dtype, cache, 16))
    i32 = dict(dtype=torch.int32, device=DEV)
    room = torch.full((rows, 3, heads, dim + 8), 7.0, dtype=dtype, device=DEV)
    lse = torch.full((rows, heads), 7.0, device=DEV)
    out = A.tree_attention(ctx, s["q"], s["cache_k"], s["cache_v"], torch.empty((0, 4), **i32), torch.empty(0, **i32),
                           torch.zeros(1, **i32), k_scale=s["k_scale"], v_scale=s["v_scale"], out=room[:, 1, :, :dim], lse=lse)
    torch.cuda.synchronize()
    assert not out.any() and (lse == -float("inf")).all()
    room[:, 1, :, :dim] = 7.0
    assert (room == 7.0).all()  # and nothing beside it
