"""Operators over paged key-value caches, on torch tensors.

A program that lays key-value caches out on the GPU with relocation plans
then attends over them. The calls of its step, in order:

  block_tables          where the step's tokens go: slots, positions, pages
                        taken from the free list, masks of drafted trees
  norm_rotate_append    norm and rotation of the step's queries and keys; keys
                        and values into the cache (int8 by a scale a head)
  block_append          or, after `norm_rotate`, keys and values into an int8
                        cache with a scale for each block of tokens and head
  tree_attention        attention of the step's rows over the cache, all of it
                        or a window with first tokens that stay

and, in training, `norm_rotate` (a differentiable function of its queries, keys
and weights) and `window_attention` over packed sequences, with
`norm_rotate_backward` and `window_attention_backward` beneath them.

Calls take a `pyreloc.Context`, run on torch's current stream of its device,
return at once and never wait for the GPU, so they can be captured into a
graph; results are fresh tensors unless `out` is given. The package's own
plans write caches that these calls read as they are: the int8 result
[requests, heads, tokens, dim] of the C5 plan is the cache
`result.transpose(1, 2)`, with one page a request. Bad arguments raise
ValueError, what the library refuses TransferError("<code>: <detail>").
"""
import ctypes
import struct
import threading
from collections import namedtuple
from functools import lru_cache, partial

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native as N
from .transfer import _fail

_KINDS = {torch.float32: (0, 32), torch.float16: (0, 16), torch.bfloat16: (1, 16), torch.int8: (2, 8)}

Tables = namedtuple("Tables", "starts slots positions taken mask")
Tables.__doc__ = """Where a step's tokens go (see `block_tables`): each request's first row
[requests + 1], and per row its slot (int64, -1: none) and position; the pages
wanted from the free list [1]; the trees' ancestor masks [rows, words] or None."""


def _format(record):
    """A record's fields as one struct format: all are eight bytes wide."""
    out = ""
    for _, t in record._fields_:
        out += _format(t) if issubclass(t, ctypes.Structure) else \
            "d" if t is ctypes.c_double else "Q" if t is ctypes.c_void_p else "q"
    return out


_HEADS = struct.Struct(_format(N.relx_heads))
_CACHE = struct.Struct(_format(N.relx_cache))
_TABLES = struct.Struct(_format(N.relx_block_tables_args))
_ROTATION = struct.Struct(_format(N.relx_rotation))
_ATTENTION = struct.Struct(_format(N.relx_tree_attention_args)[6:])  # after its two relx_heads
_SCALES = struct.Struct(_format(N.relx_block_scales))
_VIEW = struct.Struct(_format(N.relx_cache_view)[:2])  # before its scales
_WINDOW = struct.Struct(_format(N.relx_window_args)[12:])  # after its four relx_heads
_APPEND = struct.Struct(_format(N.relx_block_append_args)[6 + 16 + 6:])  # after its heads, cache and scales


def _bad(message):
    raise ValueError(message)


_functions = {}
_errors = threading.local()


def _call(name, ctx, *args):
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(N.lib(), name)
    try:
        err = _errors.err
    except AttributeError:
        err = _errors.err = N.relx_err()
        _errors.ref = ctypes.byref(err)
    if fn(ctx._h, *args, _errors.ref):
        _fail(err)


_split = torch.unsafe_split_with_sizes  # of buffers that nobody else has
# torch's current stream as a handle; the plain query costs as much as a launch
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _device(ctx, like):
    """The context's device, which every tensor of the call is on."""
    if like.get_device() != ctx.device:
        _bad("the tensors are on %s, the context on device %d" % (like.device, ctx.device))
    return ctx.device


def _row(t, name, dtype, n, device):
    """A contiguous vector of `n` (None: any number)."""
    if t.dtype is not dtype or t.get_device() != device or (t.dim() != 1 if n is None else t.shape != (n,)) or \
            not t.is_contiguous():
        _bad("%s: %s [%s] on device %d, contiguous; got %s %s on %s"
             % (name, dtype, "n" if n is None else n, device, t.dtype, list(t.shape), t.device))
    return t.data_ptr()


def _heads(t, name, shape, dtype, device):
    """[rows, heads, dim] with a contiguous last dimension, packed."""
    if t.shape != shape or t.dtype is not dtype or t.get_device() != device:
        _bad("%s: %s %s on device %d; got %s %s on %s"
             % (name, dtype, list(shape), device, t.dtype, list(t.shape), t.device))
    row, head, one = t.stride()
    if one != 1 and shape[2] > 1 and t.numel():
        _bad("%s: the last dimension must be contiguous" % name)
    return _HEADS.pack(t.data_ptr(), row, head)


def _made(t, shape):
    """A record of a tensor that the call has made, [rows, heads, dim]."""
    return _HEADS.pack(t.data_ptr(), shape[1] * shape[2], shape[2])


def _table(t, device):
    if t.dtype is not torch.int32 or t.dim() != 2 or t.get_device() != device or \
            (t.stride(1) != 1 and t.numel() > 1 and t.shape[1] > 1):
        _bad("block table: int32 [requests, columns] on device %d with contiguous rows; got %s %s on %s"
             % (device, t.dtype, list(t.shape), t.device))
    requests, columns = t.shape
    return requests, columns, t.data_ptr(), t.stride(0)


def _block_scales(k_scale, v_scale, shape, device):
    """The record of an int8 cache's scales [pages, page / block, kv_heads]."""
    kss = k_scale.shape
    if v_scale is None or v_scale.shape != kss or k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32 or \
            k_scale.get_device() != device or v_scale.get_device() != device or len(shape) != 4 or len(kss) != 3 or \
            kss[0] != shape[0] or kss[2] != shape[2] or kss[1] < 1 or shape[1] % kss[1] or k_scale.stride() != v_scale.stride():
        _bad("scales of blocks: float32 [pages, page / block, kv_heads] on device %d, alike in both; got %s %s and %s for a cache %s"
             % (device, k_scale.dtype, list(kss), "none" if v_scale is None else "%s %s" % (v_scale.dtype, list(v_scale.shape)),
                list(shape)))
    return _SCALES.pack(k_scale.data_ptr(), v_scale.data_ptr(), *k_scale.stride(), shape[1] // kss[1])


_NO_SCALES = _SCALES.pack(*(0,) * 6)


def _cache(keys, values, k_scale, v_scale, device, blocks=False):
    """The cache's record fields: keys and values [pages, page, kv_heads, dim].
    `blocks`: its scales are of blocks, in a record of their own."""
    shape, dtype = keys.shape, keys.dtype
    kind = _KINDS.get(dtype)
    if len(shape) != 4 or values.shape != shape or values.dtype is not dtype or kind is None or \
            keys.get_device() != device or values.get_device() != device:
        _bad("cache: keys and values [pages, page, kv_heads, dim] of one type on device %d; got %s %s on %s and %s %s on %s"
             % (device, dtype, list(shape), keys.device, values.dtype, list(values.shape), values.device))
    kp, ks, kh, ko = keys.stride()
    vp, vs, vh, vo = values.stride()
    if (ko != 1 or vo != 1) and shape[3] > 1 and keys.numel():
        _bad("cache: the last dimension must be contiguous")
    k_ptr = v_ptr = 0
    if blocks:
        if dtype is not torch.int8:
            _bad("scales go with an int8 cache")
        k_ptr, v_ptr = k_scale.data_ptr(), v_scale.data_ptr()
    elif dtype is torch.int8:
        if k_scale is None or v_scale is None:
            _bad("an int8 cache takes k_scale and v_scale")
        k_ptr = _row(k_scale, "k_scale", torch.float32, shape[2], device)
        v_ptr = _row(v_scale, "v_scale", torch.float32, shape[2], device)
    elif k_scale is not None or v_scale is not None:
        _bad("scales go with an int8 cache")
    return (keys.data_ptr(), kp, ks, kh, values.data_ptr(), vp, vs, vh, k_ptr, v_ptr, *shape, *kind)


def _in_graph(*operands):
    """Whether torch would follow a gradient through a call of these."""
    if torch.is_grad_enabled():
        for t in operands:
            if t is not None and t.requires_grad:
                return True
    return False


def _no_tangent(name, *operands):
    """Refuses what carries a forward-mode derivative: the result would have none,
    which says that it is zero."""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        for t in operands:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("sym_amd.attention.%s has no forward-mode derivative" % name)


class _NoGradient(torch.autograd.Function):
    """A call that has no gradient, of operands that want one: its result says so
    when a gradient reaches it, rather than end it in silence."""
    @staticmethod
    def forward(fn, name, call, *operands):
        fn.name = name
        return call()

    @staticmethod
    def backward(fn, *gradients):
        raise RuntimeError("sym_amd.attention.%s has no gradient" % fn.name)


# ------------------------------------------------------------ block tables

def block_tables(ctx, cached, fresh, table, free_pages, page, rows, *, parents=None, words=1, out=None):
    """Slots, positions and pages of a step's new tokens, on the GPU.

    Request b has `cached[b]` tokens in the cache and adds `fresh[b]` (int32
    [requests]). Pages of `page` slots are listed in `table` (int32
    [requests, columns]); the further ones that a request needs are taken from
    `free_pages` (int32) in request order and written into `table`. The step
    has `rows` rows at most (rows past the requests' get slot -1). `parents`
    (int32 [rows]) makes each request's new tokens a drafted tree: the one of
    the same request that a token follows, always an earlier one, or -1; then
    positions are those in the tree and `mask` (int64 [rows, words]) has each
    token's ancestors and itself. Returns `Tables`; `out`: such a tuple to
    write into. `taken` past len(free_pages) says that the list ran out, and
    the slots without a page are -1."""
    device = _device(ctx, table)
    requests, columns, t_ptr, t_row = _table(table, device)
    rows, page = int(rows), int(page)
    if rows < 0 or page < 1:
        _bad("block tables: rows = %d, page = %d" % (rows, page))
    c_ptr = _row(cached, "cached", torch.int32, requests, device)
    f_ptr = _row(fresh, "fresh", torch.int32, requests, device)
    l_ptr = _row(free_pages, "free_pages", torch.int32, None, device)
    if parents is None:
        words = p_ptr = 0
    else:
        words = int(words)
        p_ptr = _row(parents, "parents", torch.int32, rows, device)
        if words < 1:
            _bad("block tables: words = %d" % words)
    if out is None:
        i32 = table.new_empty(requests + 2 + rows)
        i64 = table.new_empty(rows * (1 + words), dtype=torch.int64)
        p32, p64 = i32.data_ptr(), i64.data_ptr()
        starts, taken, positions = _split(i32, (requests + 1, 1, rows))
        ptrs = p32, p64, p32 + 4 * (requests + 2), p64 + 8 * rows if words else 0, p32 + 4 * (requests + 1)
        mask = None
        if words:
            i64, mask = _split(i64, (rows, rows * words))
            mask = mask.view(rows, words)
        out = Tables(starts, i64, positions, taken, mask)
    else:
        ptrs = (_row(out.starts, "starts", torch.int32, requests + 1, device),
                _row(out.slots, "slots", torch.int64, rows, device),
                _row(out.positions, "positions", torch.int32, rows, device), 0,
                _row(out.taken, "taken", torch.int32, 1, device))
        if words:
            m = out.mask
            if m is None or m.dtype is not torch.int64 or m.shape != (rows, words) or m.get_device() != device or \
                    not m.is_contiguous():
                _bad("mask: contiguous int64 [%d, %d]" % (rows, words))
            ptrs = ptrs[:3] + (m.data_ptr(), ptrs[4])
    _call("relx_block_tables", ctx,
          _TABLES.pack(c_ptr, f_ptr, t_ptr, t_row, l_ptr, free_pages.shape[0], p_ptr, *ptrs, requests, columns, page,
                       rows, words), _stream(device))
    return out


# --------------------------------------------------------- norm and rotation

def _rotation(ctx, q, k, positions, cos, sin, q_weight, k_weight, eps, pairs):
    """(packed rotation, query and key shapes, device)."""
    device = _device(ctx, q)
    qs, ks = q.shape, k.shape
    kind = _KINDS.get(q.dtype)
    if len(qs) != 3 or len(ks) != 3 or qs[0] != ks[0] or qs[2] != ks[2] or kind is None or kind[1] == 8:
        _bad("queries [rows, heads, dim] and keys [rows, kv_heads, dim] of one floating type; got %s %s and %s %s"
             % (q.dtype, list(qs), k.dtype, list(ks)))
    rows, dim = qs[0], qs[2]
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or \
            cos.get_device() != device or sin.get_device() != device or not (cos.is_contiguous() and sin.is_contiguous()):
        _bad("cos and sin: contiguous float32 [angles, rotary / 2] on device %d; got %s %s and %s %s"
             % (device, cos.dtype, list(cos.shape), sin.dtype, list(sin.shape)))
    qw_ptr = kw_ptr = 0
    given = k_weight if q_weight is None else q_weight
    if given is None:
        w_kind = 0, 32
    else:
        w_kind = _KINDS.get(given.dtype)
        if w_kind is None or w_kind[1] == 8:
            _bad("weights: a floating type; got %s" % given.dtype)
        if q_weight is not None:
            qw_ptr = _row(q_weight, "weight", given.dtype, dim, device)
        if k_weight is not None:
            kw_ptr = _row(k_weight, "weight", given.dtype, dim, device)
    p_ptr = _row(positions, "positions", torch.int32, rows, device)
    return (_ROTATION.pack(p_ptr, cos.data_ptr(), sin.data_ptr(), qw_ptr, kw_ptr, *w_kind, rows, qs[1], ks[1], dim,
                           2 * cos.shape[1], 1 if pairs else 0, cos.shape[0], *kind, float(eps)), qs, ks, device)


class _NormRotate(torch.autograd.Function):
    @staticmethod
    def forward(fn, q, k, q_weight, k_weight, ctx, positions, cos, sin, eps, pairs):
        fn.save_for_backward(q, k, q_weight, k_weight, positions, cos, sin)
        fn.rest = ctx, eps, pairs
        return _norm_rotate(ctx, q, k, positions, cos, sin, q_weight, k_weight, eps, pairs, None)

    @staticmethod
    @once_differentiable
    def backward(fn, dq, dk):
        if fn.needs_input_grad[6] or fn.needs_input_grad[7]:
            raise RuntimeError("sym_amd.attention.norm_rotate has no gradient for cos and sin")
        q, k, q_weight, k_weight, positions, cos, sin = fn.saved_tensors
        ctx, eps, pairs = fn.rest
        gq, gk, gqw, gkw = norm_rotate_backward(ctx, dq.contiguous(), dk.contiguous(), q, k, positions, cos, sin,
                                                q_weight, k_weight, eps, pairs=pairs,
                                                weight_grads=fn.needs_input_grad[2:4])
        return (gq, gk, None if gqw is None else gqw.to(q_weight.dtype),
                None if gkw is None else gkw.to(k_weight.dtype), None, None, None, None, None, None)


def norm_rotate(ctx, q, k, positions, cos, sin, q_weight, k_weight, eps, *, pairs=False, out=None):
    """Root-mean-square norm of each head, times a weight [dim] (None: 1), then
    the rotation by position, in one pass over the queries [rows, heads, dim]
    and keys [rows, kv_heads, dim] (f32, f16 or bf16; any row and head strides,
    so views of a fused projection do).

    `positions` (int32 [rows]) index `cos` and `sin` (float32
    [angles, rotary / 2]), which turn the first `rotary` elements: halves
    (i, i + rotary / 2), or neighbours (2 i, 2 i + 1) with `pairs`. A position
    outside the table gives NaN. Returns (queries, keys); `out`: a pair of
    tensors to write into. Differentiable in q, k and the weights, once (without
    `out`; a second derivative, one by cos and sin, or one of forward mode raises)."""
    _no_tangent("norm_rotate", q, k, q_weight, k_weight, cos, sin)
    if out is None and _in_graph(q, k, q_weight, k_weight, cos, sin):
        return _NormRotate.apply(q, k, q_weight, k_weight, ctx, positions, cos, sin, eps, pairs)
    return _norm_rotate(ctx, q, k, positions, cos, sin, q_weight, k_weight, eps, pairs, out)


def _norm_rotate(ctx, q, k, positions, cos, sin, q_weight, k_weight, eps, pairs, out):
    rot, qs, ks, device = _rotation(ctx, q, k, positions, cos, sin, q_weight, k_weight, eps, pairs)
    dtype = q.dtype
    if out is None:
        zq, zk = q.new_empty(qs), k.new_empty(ks)
        results = _made(zq, qs), _made(zk, ks)
    else:
        zq, zk = out
        results = _heads(zq, "query result", qs, dtype, device), _heads(zk, "key result", ks, dtype, device)
    _call("relx_norm_rotate", ctx, rot, _heads(q, "queries", qs, dtype, device), _heads(k, "keys", ks, dtype, device),
          *results, _stream(device))
    return zq, zk


def norm_rotate_backward(ctx, dq, dk, q, k, positions, cos, sin, q_weight, k_weight, eps, *, pairs=False,
                         weight_grads=(True, True)):
    """Gradients of `norm_rotate` for its results' gradients `dq` and `dk`:
    (queries', keys', query weight's, key weight's). The weights' are float32
    [dim], summed over rows and heads in a fixed order (None where the weight
    is, or where `weight_grads` says that it is not wanted); the others have the
    operands' type."""
    _no_tangent("norm_rotate_backward", dq, dk, q, k, q_weight, k_weight, cos, sin)
    rot, qs, ks, device = _rotation(ctx, q, k, positions, cos, sin, q_weight, k_weight, eps, pairs)
    dtype = q.dtype
    gq, gk = q.new_empty(qs), k.new_empty(ks)
    gqw = gkw = None
    gqw_ptr = gkw_ptr = room_ptr = size = 0
    if q_weight is not None and weight_grads[0]:
        gqw = cos.new_empty(qs[2])
        gqw_ptr = gqw.data_ptr()
    if k_weight is not None and weight_grads[1]:
        gkw = cos.new_empty(qs[2])
        gkw_ptr = gkw.data_ptr()
    if gqw_ptr or gkw_ptr:
        size = _rotate_room(rot, qs, ks, dtype)
        room = cos.new_empty(size // 4)
        room_ptr = room.data_ptr()
    _call("relx_norm_rotate_backward", ctx, rot, _heads(dq, "query gradient", qs, dtype, device),
          _heads(dk, "key gradient", ks, dtype, device), _heads(q, "queries", qs, dtype, device),
          _heads(k, "keys", ks, dtype, device), _made(gq, qs), _made(gk, ks), gqw_ptr, gkw_ptr, room_ptr, size, _stream(device))
    return gq, gk, gqw, gkw


_rooms = {}


def _rotate_room(rot, qs, ks, dtype):
    # other threads may clear the sizes at any time
    key = (qs, ks[1], dtype)
    room = _rooms.get(key)
    if room is None:
        size, err = ctypes.c_size_t(), N.relx_err()
        if N.lib().relx_norm_rotate_workspace(rot, ctypes.byref(size), ctypes.byref(err)):
            _fail(err)
        room = size.value
        if len(_rooms) >= 1024:
            _rooms.clear()
        _rooms[key] = room
    return room


def norm_rotate_append(ctx, q, k, v, slots, cache_k, cache_v, positions, cos, sin, q_weight, k_weight, eps, *,
                       pairs=False, k_scale=None, v_scale=None, out=None):
    """The serving form of `norm_rotate`: returns the queries (in `out`, which
    may be `q` itself), and puts the keys, and the values `v` [rows, kv_heads,
    dim] as they are, into the cache at each row's slot (int64 [rows]; a slot
    outside the cache is skipped, and rows have slots of their own). The cache
    is [pages, page, kv_heads, dim] of any strides, of the operands' type, or
    int8 with a scale a head (float32 [kv_heads] each), quantized as the
    package's plans quantize. There is no gradient: one that reaches the result
    (without `out`) raises."""
    _no_tangent("norm_rotate_append", q, k, v, cos, sin, q_weight, k_weight)
    if out is None and _in_graph(q, k, v, cos, sin, q_weight, k_weight):
        return _NoGradient.apply(
            "norm_rotate_append",
            partial(norm_rotate_append, ctx, q, k, v, slots, cache_k, cache_v, positions, cos, sin, q_weight, k_weight, eps,
                    pairs=pairs, k_scale=k_scale, v_scale=v_scale), q, k, v, cos, sin, q_weight, k_weight)
    rot, qs, ks, device = _rotation(ctx, q, k, positions, cos, sin, q_weight, k_weight, eps, pairs)
    dtype = q.dtype
    if out is None:
        out = q.new_empty(qs)
        result = _made(out, qs)
    else:
        result = _heads(out, "query result", qs, dtype, device)
    cache = _CACHE.pack(*_cache(cache_k, cache_v, k_scale, v_scale, device))
    _call("relx_norm_rotate_append", ctx, rot, _heads(q, "queries", qs, dtype, device),
          _heads(k, "keys", ks, dtype, device), _heads(v, "values", ks, dtype, device),
          result, _row(slots, "slots", torch.int64, qs[0], device),
          cache, _stream(device))
    return out


# ------------------------------------------------------------ blocks of a cache

def block_append(ctx, k, v, cache_k, cache_v, k_scale, v_scale, table, cached, starts):
    """Quantizes a step's keys and values [rows, kv_heads, dim] (f32, f16 or bf16,
    any row and head strides) into an int8 cache [pages, page, kv_heads, dim] whose
    blocks of tokens have a scale each for every head: `k_scale` and `v_scale`,
    float32 [pages, page / block, kv_heads] of any strides, the same in both, with
    blocks of a multiple of 16 tokens.

    Request b's rows [starts[b], starts[b + 1]) become the tokens cached[b], ... of
    its row of `table` (int32 [requests, columns]). A block's scale is the largest
    finite magnitude of its tokens / 127: where it grows, the codes of the tokens
    that the request already has in the block are rounded anew. Infinities become
    the largest codes, NaN -128, as in the package's plans. Tokens whose page is
    not in the cache are left out; a block is of one request that writes to it.
    Caches and scales are updated in place; there is no gradient, so keys or values
    that want one are refused (in a graph, detach them)."""
    _no_tangent("block_append", k, v)
    if _in_graph(k, v):
        _bad("block_append has no gradient: it takes detached keys and values, or runs under torch.no_grad()")
    device = _device(ctx, k)
    shape, dtype = k.shape, k.dtype
    kind = _KINDS.get(dtype)
    if len(shape) != 3 or kind is None or kind[1] == 8 or cache_k.dim() != 4 or cache_k.dtype is not torch.int8 or \
            cache_k.shape[2:] != shape[1:]:
        _bad("keys: a floating type [rows, kv_heads, dim], into an int8 cache of the same heads; got %s %s and %s %s"
             % (dtype, list(shape), cache_k.dtype, list(cache_k.shape)))
    scales = _block_scales(k_scale, v_scale, cache_k.shape, device)
    requests, columns, t_ptr, t_row = _table(table, device)
    _call("relx_block_append", ctx,
          _heads(k, "keys", shape, dtype, device) + _heads(v, "values", shape, dtype, device) +
          _CACHE.pack(*_cache(cache_k, cache_v, k_scale, v_scale, device, True)) + scales +
          _APPEND.pack(t_ptr, t_row, _row(cached, "cached", torch.int32, requests, device),
                       _row(starts, "starts", torch.int32, requests + 1, device), shape[0], requests, columns, *kind),
          _stream(device))


# ------------------------------------------------------------ attention

@lru_cache(maxsize=4096)
def tree_attention_workspace(rows, requests, heads, kv_heads, dim, page):
    """Bytes of device memory that a `tree_attention` call of these sizes
    works in. They go by rows / requests, so fewer rows may take more: the bytes
    of all rows in one request, and eight a request, are enough for every call of
    at most so many rows and requests."""
    size, err = ctypes.c_size_t(), N.relx_err()
    args = N.relx_tree_attention_args()
    args.rows, args.requests, args.heads = rows, requests, heads
    args.cache.kv_heads, args.cache.dim, args.cache.page = kv_heads, dim, page
    if N.lib().relx_tree_attention_workspace(bytes(args), ctypes.byref(size), ctypes.byref(err)):
        _fail(err)
    return size.value


def tree_attention(ctx, q, cache_k, cache_v, table, cached, starts, *, mask=None, scale=None, k_scale=None,
                   v_scale=None, window=None, sinks=0, out=None, lse=None, workspace=None):
    """Attention of a step's rows q [rows, heads, dim] (f16, bf16) over a paged
    cache [pages, page, kv_heads, dim] of any strides, of the same type or
    int8 with scales [kv_heads].

    Request b has the rows [starts[b], starts[b + 1]) and sees the `cached[b]`
    first tokens of its row of `table`, and of its own new ones, which are
    already in the cache after them, those whose bit its row of `mask` (int64
    [rows, words], as `block_tables` makes it) has; without a mask, those up to
    itself (one row a request: plain decoding). Head h reads key head
    h // (heads // kv_heads). A row that sees nothing, or of no request, is 0.

    `window` (None or 0: of everything): a row at position p sees of the tokens x
    only those with p - x < window, and the first `sinks` ones; p is cached + j, or with a mask
    cached + the token's depth in its tree, of which it sees what its mask says
    (the window has to hold the tree: 64 * words at least). An int8 cache
    with a scale a block of tokens, as `block_append` fills it, has scales
    [pages, page / block, kv_heads] (float32, any strides, the same in both).

    `scale`: of the scores, by default dim ** -0.5. `lse`: float32 [rows,
    heads] for the logarithm of each row's sum of exponentials. `workspace`: a
    uint8 tensor of `tree_attention_workspace` bytes, for programs that keep
    one a stream; by default torch's allocator gives it. There is no gradient:
    one that reaches the result (without `out`) raises."""
    _no_tangent("tree_attention", q, cache_k, cache_v, k_scale, v_scale)
    if out is None and _in_graph(q, cache_k, cache_v, k_scale, v_scale):
        return _NoGradient.apply(
            "tree_attention",
            partial(tree_attention, ctx, q, cache_k, cache_v, table, cached, starts, mask=mask, scale=scale, k_scale=k_scale,
                    v_scale=v_scale, window=window, sinks=sinks, lse=lse, workspace=workspace), q, cache_k, cache_v, k_scale,
            v_scale)
    device = _device(ctx, q)
    shape, dtype = q.shape, q.dtype
    kind = _KINDS.get(dtype)
    if len(shape) != 3 or kind is None or kind[1] != 16:
        _bad("queries: f16 or bf16 [rows, heads, dim]; got %s %s" % (dtype, list(shape)))
    rows, heads, dim = shape
    blocks = k_scale is not None and k_scale.dim() == 3
    scales = _block_scales(k_scale, v_scale, cache_k.shape, device) if blocks else _NO_SCALES
    cache = _cache(cache_k, cache_v, k_scale, v_scale, device, blocks)
    kv_heads = cache[12]
    if cache[13] != dim or kv_heads < 1 or heads < 1 or heads % kv_heads or \
            (cache_k.dtype is not dtype and cache_k.dtype is not torch.int8):
        _bad("cache: %s or int8 [pages, page, kv_heads, %d] with kv_heads dividing %d; got %s %s"
             % (dtype, dim, heads, cache_k.dtype, list(cache_k.shape)))
    requests, columns, t_ptr, t_row = _table(table, device)
    words = m_ptr = 0
    if mask is not None:
        if mask.dtype is not torch.int64 or mask.dim() != 2 or mask.shape[0] != rows or mask.get_device() != device or \
                not mask.is_contiguous() or mask.shape[1] < 1:
            _bad("mask: contiguous int64 [%d, words] on device %d; got %s %s" % (rows, device, mask.dtype, list(mask.shape)))
        words, m_ptr = mask.shape[1], mask.data_ptr()
    if out is None:
        out = q.new_empty(shape)
        result = _made(out, shape)
    else:
        result = _heads(out, "result", shape, dtype, device)
    l_ptr = 0
    if lse is not None:
        if lse.dtype is not torch.float32 or lse.shape != shape[:2] or lse.get_device() != device or not lse.is_contiguous():
            _bad("lse: contiguous float32 [%d, %d]" % (rows, heads))
        l_ptr = lse.data_ptr()
    if workspace is None:
        workspace = q.new_empty(tree_attention_workspace(rows, requests, heads, kv_heads, dim, cache[11]),
                                dtype=torch.uint8)
    elif workspace.dtype is not torch.uint8 or workspace.get_device() != device or not workspace.is_contiguous():
        _bad("workspace: contiguous uint8 on device %d" % device)
    args = _heads(q, "queries", shape, dtype, device) + result + \
        _ATTENTION.pack(*cache, t_ptr, t_row, _row(cached, "cached", torch.int32, requests, device),
                        _row(starts, "starts", torch.int32, requests + 1, device), m_ptr, l_ptr,
                        workspace.data_ptr(), workspace.numel(), rows, requests, heads, columns, words, *kind,
                        dim ** -0.5 if scale is None else float(scale))
    if window is None and not blocks:
        if sinks:
            _bad("first tokens that stay go with a window")
        _call("relx_tree_attention", ctx, args, _stream(device))
    else:
        _call("relx_tree_attention_view", ctx, args, _view(window, sinks) + scales, _stream(device))
    return out


def _reach(window, sinks):
    """Both as the library takes them: whole numbers of 63 bits, no window as 0."""
    window, sinks = 0 if window is None else int(window), int(sinks)
    if window < 0 or sinks < 0 or (window == 0 and sinks):
        _bad("a window of %d tokens with %d first ones" % (window, sinks))
    return min(window, 1 << 62), min(sinks, 1 << 62)


def _view(window, sinks):
    return _VIEW.pack(*_reach(window, sinks))


# ------------------------------------------------------------ packed sequences

class _Window(torch.autograd.Function):
    @staticmethod
    def forward(fn, q, k, v, ctx, starts, window, sinks, scale, lse):
        # the backward's own: the caller's buffer may be another call's before that runs
        own = q.new_empty((q.shape[1], q.shape[0]), dtype=torch.float32) if lse is None else lse
        out = _window_attention(ctx, q, k, v, starts, window, sinks, scale, None, own)
        fn.save_for_backward(q, k, v, out, own if lse is None else lse.clone(), starts)
        fn.rest = ctx, window, sinks, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(fn, dout):
        q, k, v, out, lse, starts = fn.saved_tensors
        ctx, window, sinks, scale = fn.rest
        dq, dk, dv = window_attention_backward(ctx, _packed(dout), q, k, v, out, lse, starts, window=window, sinks=sinks, scale=scale)
        wants = fn.needs_input_grad
        return dq if wants[0] else None, dk if wants[1] else None, dv if wants[2] else None, None, None, None, None, None, None


def _packed(t):
    """A gradient as it lies, if its rows do as the kernels want them, or a copy: one
    whose elements lie in order may begin at any address."""
    row, head, one = t.stride()
    if one == 1 and row % 8 == 0 and head % 8 == 0 and 0 < row <= 1 << 24 and head > 0 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _window_record(ctx, q, k, v, out, lse, starts, window, sinks, scale):
    device = _device(ctx, q)
    shape, ks, dtype = q.shape, k.shape, q.dtype
    kind = _KINDS.get(dtype)
    if len(shape) != 3 or len(ks) != 3 or kind is None or kind[1] != 16 or ks[0] != shape[0] or ks[2] != shape[2] or \
            ks[1] < 1 or shape[1] < 1 or shape[1] % ks[1]:
        _bad("queries and keys: f16 or bf16 [rows, heads, dim] and [rows, kv_heads, dim], kv_heads dividing heads; got %s %s and %s %s"
             % (dtype, list(shape), k.dtype, list(ks)))
    window, sinks = _reach(window, sinks)
    l_ptr = 0
    if lse is not None:
        if lse.dtype is not torch.float32 or lse.shape != (shape[1], shape[0]) or lse.get_device() != device or \
                not lse.is_contiguous():
            _bad("lse: contiguous float32 [%d, %d]" % (shape[1], shape[0]))
        l_ptr = lse.data_ptr()
    if starts.dim() != 1 or starts.shape[0] < 1:
        _bad("starts: int32 [sequences + 1]")
    return (_heads(q, "queries", shape, dtype, device) + _heads(k, "keys", ks, dtype, device) +
            _heads(v, "values", ks, dtype, device) + _heads(out, "result", shape, dtype, device) +
            _WINDOW.pack(_row(starts, "starts", torch.int32, None, device), l_ptr, shape[0], starts.shape[0] - 1, shape[1], ks[1],
                         shape[2], window, sinks, *kind, shape[2] ** -0.5 if scale is None else float(scale))), device


def window_attention(ctx, q, k, v, starts, *, window=None, sinks=0, scale=None, out=None, lse=None):
    """Attention over packed sequences, for training and prompts: sequence b has the
    rows [starts[b], starts[b + 1]) (int32 [sequences + 1]) of the queries
    [rows, heads, dim] and of the keys and values [rows, kv_heads, dim] (f16 or bf16;
    strides of multiples of eight elements, so views of a fused projection do). Head h
    reads key head h // (heads // kv_heads).

    A row at place p of its sequence sees the places x <= p with p - x < `window`
    (None or 0: any), and the first `sinks` ones (256 at most, unless no row leaves the
    window). Rows of no sequence are
    0, and nothing of one sequence reaches another. `scale`: of the scores, by
    default dim ** -0.5. `lse`: float32 [heads, rows] for the logarithm of each row's
    sum of exponentials. Differentiable in q, k and v, once (without `out`; a second
    derivative, or one of forward mode, raises)."""
    _no_tangent("window_attention", q, k, v)
    if out is None and _in_graph(q, k, v):
        return _Window.apply(q, k, v, ctx, starts, window, sinks, scale, lse)
    return _window_attention(ctx, q, k, v, starts, window, sinks, scale, out, lse)


def _window_attention(ctx, q, k, v, starts, window, sinks, scale, out, lse):
    if out is None:
        out = q.new_empty(q.shape)
    args, device = _window_record(ctx, q, k, v, out, lse, starts, window, sinks, scale)
    _call("relx_window_attention", ctx, args, _stream(device))
    return out


def window_attention_backward(ctx, dout, q, k, v, out, lse, starts, *, window=None, sinks=0, scale=None):
    """Gradients of `window_attention` for its result's gradient `dout`, from its
    result and its `lse`: (queries', keys', values'), of the operands' type; those of
    keys and values are summed over a key head's query heads. The same bits every time."""
    _no_tangent("window_attention_backward", dout, q, k, v, out, lse)
    args, device = _window_record(ctx, q, k, v, out, lse, starts, window, sinks, scale)
    if lse is None:
        _bad("the backward takes the forward's lse")
    shape, ks = q.shape, k.shape
    dq, dk, dv = q.new_empty(shape), q.new_empty(ks), q.new_empty(ks)
    size = _window_room(args, shape, ks, q.dtype, starts.shape[0], window, sinks)
    room = q.new_empty(size, dtype=torch.uint8)
    _call("relx_window_attention_backward", ctx, args, _heads(dout, "result's gradient", shape, q.dtype, device),
          _made(dq, shape), _made(dk, ks), _made(dv, ks), room.data_ptr(), size, _stream(device))
    return dq, dk, dv


def _window_room(args, shape, ks, dtype, starts, window, sinks):
    key = (shape, ks[1], dtype, starts, window, sinks)
    room = _rooms.get(key)
    if room is None:
        size, err = ctypes.c_size_t(), N.relx_err()
        if N.lib().relx_window_attention_workspace(args, ctypes.byref(size), ctypes.byref(err)):
            _fail(err)
        room = size.value
        if len(_rooms) >= 1024:
            _rooms.clear()
        _rooms[key] = room
    return room
