"""The paged-cache operators' boundary, without a GPU: the records that cross it,
and what the library refuses before it looks at a device."""
import ctypes
import os
import random
import re
import struct

import pytest

from tests import attention_cases as C

torch = pytest.importorskip("torch")
from sym_amd import _native as N  # noqa: E402
from sym_amd import attention as A  # noqa: E402

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "relx.h")
RECORDS = ["relx_heads", "relx_cache", "relx_block_tables_args", "relx_rotation", "relx_tree_attention_args"]


@pytest.fixture(scope="module")
def lib():
    return N.lib()


def refused(fn, *args):
    err = N.relx_err()
    assert fn(*args, ctypes.byref(err)) != 0
    return err.code.decode()


def test_records_are_the_headers():
    """Every field of the header's records, in its order, eight bytes each."""
    text = open(HEADER).read()
    for name in RECORDS:
        body = re.sub(r"/\*.*?\*/|//[^\n]*", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1),
                      flags=re.S)
        fields = []
        for line in body.split(";"):
            line = line.strip()
            if line:
                fields += [re.sub(r"\W", "", part.split()[-1]) for part in line.split(",")]
        record = getattr(N, name)
        assert [f for f, _ in record._fields_] == fields, name
        flat = struct.Struct(A._format(record))
        assert flat.size == ctypes.sizeof(record) == 8 * len(A._format(record))


def test_workspace_sizes(lib):
    a = A.tree_attention_workspace(8, 8, 32, 8, 128, 16)
    assert 0 < a < A.tree_attention_workspace(8 * 64, 8, 32, 8, 128, 16) < 1 << 30
    size = ctypes.c_size_t()
    for bad in (dict(rows=-1), dict(requests=-1), dict(heads=0), dict(page=0), dict(kv_heads=0)):
        args = N.relx_tree_attention_args()
        args.rows = args.requests = args.heads = 1
        args.cache.kv_heads = args.cache.dim = args.cache.page = 1
        for k, v in bad.items():
            setattr(args if hasattr(args, k) else args.cache, k, v)
        assert refused(lib.relx_tree_attention_workspace, bytes(args), ctypes.byref(size)) == "invalid_argument", bad


def test_null_arguments(lib):
    size = ctypes.c_size_t()
    assert refused(lib.relx_block_tables, None, None, 0) == "invalid_argument"
    assert refused(lib.relx_tree_attention, None, None, 0) == "invalid_argument"
    assert refused(lib.relx_tree_attention_workspace, None, ctypes.byref(size)) == "invalid_argument"
    assert refused(lib.relx_norm_rotate_workspace, None, ctypes.byref(size)) == "invalid_argument"
    assert refused(lib.relx_norm_rotate, None, None, None, None, None, None, 0) == "invalid_argument"


def test_a_context_is_needed(lib):
    args = N.relx_block_tables_args()
    args.page = 16
    assert refused(lib.relx_block_tables, None, bytes(args), 0) == "invalid_argument"


@pytest.mark.parametrize("bad", [dict(requests=-1), dict(rows=2 ** 31), dict(columns=-1), dict(page=0), dict(free_count=-1),
                                 dict(requests=1)])
def test_block_tables_refuses(lib, bad):
    args = N.relx_block_tables_args()
    args.page = 16
    for k, v in bad.items():
        setattr(args, k, v)
    assert refused(lib.relx_block_tables, None, bytes(args), 0) == "invalid_argument"


def test_tensors_that_are_not_on_the_contexts_device():
    class Other:
        device = 0
    z = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="device"):
        A.block_tables(Other, z, z, torch.zeros((1, 1), dtype=torch.int32), z, 16, 1)
    h = torch.zeros((1, 1, 8), dtype=torch.float16)
    with pytest.raises(ValueError, match="device"):
        A.norm_rotate(Other, h, h, z, torch.zeros((1, 4)), torch.zeros((1, 4)), None, None, 1e-6)
    with pytest.raises(ValueError, match="device"):
        A.tree_attention(Other, h, h[None], h[None], z[None], z, z)


def test_the_gradients_formula_against_differences():
    gen = torch.Generator().manual_seed(5)
    x, dz = (torch.randn((3, 2, 12), generator=gen, dtype=torch.float64) for _ in range(2))
    w = torch.rand(12, generator=gen, dtype=torch.float64) + 0.5
    angle = torch.rand((3, 4), generator=gen, dtype=torch.float64) * 6
    for pairs in (False, True):
        def value(x, w):
            return float((C.norm_rotate(x, w, angle.cos(), angle.sin(), 8, pairs, 1e-3)[0] * dz).sum())
        dx, _, dw, _ = C.norm_rotate_back(dz, x, w, angle.cos(), angle.sin(), 8, pairs, 1e-3)
        rng, h = random.Random(1), 1e-5
        for _ in range(20):
            i = tuple(rng.randrange(n) for n in x.shape)
            d = torch.zeros_like(x)
            d[i] = h
            assert abs((value(x + d, w) - value(x - d, w)) / (2 * h) - float(dx[i])) < 1e-8
            d = torch.zeros_like(w)
            d[i[2]] = h
            assert abs((value(x, w + d) - value(x, w - d)) / (2 * h) - float(dw[i[2]])) < 1e-8
