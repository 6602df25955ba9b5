"""Plain 64-bit forms of the paged-cache operators, and inputs for them."""
import random

import numpy as np
import torch

ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
F32 = 2.0 ** -24  # the kernels compute in 32 bits: relative error of one operation


# ------------------------------------------------------------ block tables

def tables(cached, fresh, table, free, page, rows, parents=None, words=0):
    """Token by token, from the definition."""
    table = [list(r) for r in table]
    columns = len(table[0]) if table else 0
    starts, slots, positions, masks, taken = [0], [], [], [], 0
    for b, (c, f) in enumerate(zip(cached, fresh)):
        c, f = max(c, 0), max(f, 0)
        have = min(columns, -(-c // page))
        wants = min(columns, -(-(c + f) // page))
        for g in range(have, wants):
            at = taken + g - have
            table[b][g] = free[at] if at < len(free) else -1
        taken += wants - have
        start = starts[-1]
        for j in range(f):
            if len(slots) >= rows:
                break
            g, off = divmod(c + j, page)
            page_id = table[b][g] if g < columns else -1
            slots.append(page_id * page + off if page_id >= 0 else -1)
            if parents is None:
                positions.append(c + j)
                continue
            chain, cur = [], j
            while cur >= 0:
                chain.append(cur)
                up = parents[start + cur]
                cur = up if up < cur else -1
            positions.append(c + len(chain) - 1)
            bits = [0] * words
            for i in chain:
                if i // 64 < words:
                    bits[i // 64] |= 1 << (i % 64)
            masks.append([w - (1 << 64) if w >> 63 else w for w in bits])
        starts.append(start + f)
    # pages that no row reached because the rows ran out are not in the table
    pad = rows - len(slots)
    return (starts, slots + [-1] * pad, positions + [0] * pad, taken, table,
            masks + [[0] * words] * pad if parents is not None else None)


# --------------------------------------------------------- norm and rotation

def turn(y, cos, sin, rotary, pairs, sign=1.0):
    """y [rows, heads, dim], cos and sin [rows, rotary / 2], all in 64 bits."""
    half = rotary // 2
    first = torch.arange(half) * 2 if pairs else torch.arange(half)
    second = first + (1 if pairs else half)
    c, s = cos[:, None, :], sign * sin[:, None, :]
    z = y.clone()
    z[..., first] = y[..., first] * c - y[..., second] * s
    z[..., second] = y[..., second] * c + y[..., first] * s
    return z


def norm(x, eps):
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return x * r, r


def norm_rotate(x, w, cos, sin, rotary, pairs, eps):
    """(result, bound of a 32-bit computation's error before its rounding)."""
    n, _ = norm(x.double(), eps)
    y = n * (1.0 if w is None else w.double())
    z = turn(y, cos, sin, rotary, pairs)
    # the norm's sum of squares is relatively exact to (dim + 4) roundings at
    # most, halved by the root; then four more
    size = turn(y.abs(), cos.abs(), -sin.abs(), rotary, pairs)
    size = torch.maximum(size.abs(), turn(y.abs(), cos.abs(), sin.abs(), rotary, pairs).abs())
    return z, (x.shape[-1] / 2 + 8) * F32 * size


def norm_rotate_back(dz, x, w, cos, sin, rotary, pairs, eps):
    """(gradient, its bound, weight gradient, sum of its terms' sizes)."""
    g = turn(dz.double(), cos, sin, rotary, pairs, -1.0)
    n, r = norm(x.double(), eps)
    u = g * (1.0 if w is None else w.double())
    mean = (u * n).mean(-1, keepdim=True)
    size = turn(dz.double().abs(), cos.abs(), sin.abs(), rotary, pairs, -1.0).abs()
    size = torch.maximum(size, turn(dz.double().abs(), cos.abs(), sin.abs(), rotary, pairs).abs())
    uu = size * (1.0 if w is None else w.double().abs())
    dim = x.shape[-1]
    bound = (1.5 * dim + 16) * F32 * r * (uu + n.abs() * (uu * n.abs()).mean(-1, keepdim=True))
    return r * (u - n * mean), bound, (g * n).sum((0, 1)), (size * n.abs()).sum((0, 1))


# ------------------------------------------------------------ attention

def visible(cached, fresh, limit, mask_rows):
    """[fresh, limit] what each row of a request sees of its tokens."""
    see = torch.zeros((fresh, limit), dtype=torch.bool)
    see[:, :min(cached, limit)] = True
    for j in range(fresh):
        for i in range(fresh):
            if cached + i >= limit:
                break
            if mask_rows is None:
                see[j, cached + i] = i <= j
            else:
                w = int(mask_rows[j][i // 64]) if i // 64 < len(mask_rows[j]) else 0
                see[j, cached + i] = bool(w >> (i % 64) & 1)
    return see


def attention(q, keys, values, table, cached, starts, mask, scale, k_scale, v_scale, round_to):
    """(result, lse, error bound), row by row in 64 bits on the CPU."""
    rows, heads, dim = q.shape
    pages, page, kv, _ = keys.shape
    out = torch.zeros((rows, heads, dim), dtype=torch.float64)
    bound = torch.zeros_like(out)
    lse = torch.full((rows, heads), -float("inf"), dtype=torch.float64)
    group, columns = heads // kv, table.shape[1]
    u = ROUND[round_to]
    for b in range(table.shape[0]):
        r0, r1 = int(starts[b]), int(starts[b + 1])
        if r1 <= r0:
            continue
        c = int(cached[b])
        limit = min(c + r1 - r0, columns * page)
        ids = table[b].long().repeat_interleave(page)[:limit]
        off = torch.arange(limit) % page
        there = (ids >= 0) & (ids < pages)
        k = keys[ids.clamp(0, pages - 1), off].double()
        v = values[ids.clamp(0, pages - 1), off].double()
        if k_scale is not None:
            k, v = k * k_scale.double()[:, None], v * v_scale.double()[:, None]
        see = visible(c, r1 - r0, limit, None if mask is None else mask[r0:r1].tolist()) & there[None, :]
        for h in range(heads):
            for j in range(r1 - r0):
                at = see[j].nonzero()[:, 0]
                if at.numel() == 0:
                    continue
                kk, vv = k[at, h // group], v[at, h // group]
                s = (kk @ q[r0 + j, h].double()) * scale
                lse[r0 + j, h] = torch.logsumexp(s, 0)
                p = torch.softmax(s, 0)
                o = p @ vv
                out[r0 + j, h] = o
                # the score in 32 bits (products and their sum, scaled): its error is the
                # weight's relative one; the weight is rounded to the result's type (f16: to
                # 2^-31 of the sum at least), the sums and the result once more
                ds = (dim + 4) * F32 * float((kk.abs() @ q[r0 + j, h].double().abs()).max()) * scale
                size = p @ vv.abs()
                steps = at.numel() / 32 + 16
                bound[r0 + j, h] = u * o.abs() + (u + 2 * ds + steps * F32) * size + \
                    at.numel() * 2.0 ** -31 * vv.abs().amax(0)
    return out, lse, bound


def page_table(rng, lengths, page, columns, spare=2):
    """Pages in no order; -1 past each request's own; and their number."""
    need = [min(columns, -(-n // page)) for n in lengths]
    ids = list(range(sum(need) + spare))
    rng.shuffle(ids)
    table = np.full((len(lengths), columns), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return torch.from_numpy(table), len(ids)


def tree(rng, n):
    return [rng.randint(max(-1, j - 5), j - 1) for j in range(n)]


def tree_mask(parents, words):
    rows = []
    for j, p in enumerate(parents):
        rows.append((1 << j) | (rows[p] if p >= 0 else 0))
    return [[((r >> (64 * w)) & (2 ** 64 - 1)) - (2 ** 64 if (r >> (64 * w + 63)) & 1 else 0) for w in range(words)]
            for r in rows]


def attention_case(seed, cached, fresh, heads, kv, dim, dtype, cache, page, order="slots", tree_words=0, columns=None,
                   std=1.0):
    """Operands on the CPU of a step of requests with these lengths."""
    rng = random.Random(seed)
    gen = torch.Generator().manual_seed(seed)
    lengths = [c + f for c, f in zip(cached, fresh)]
    columns = max(-(-n // page) for n in lengths) + 1 if columns is None else columns
    table, pages = page_table(rng, lengths, page, columns)
    shape = (pages, page, kv, dim) if order == "slots" else (pages, kv, page, dim)
    if cache == torch.int8:
        made = [torch.randint(-127, 128, shape, generator=gen, dtype=torch.int8) for _ in range(2)]
        scales = [torch.rand(kv, generator=gen) * 0.02 + 0.005 for _ in range(2)]
    else:
        made = [(torch.randn(shape, generator=gen) * std).to(cache) for _ in range(2)]
        scales = [None, None]
    if order == "heads":
        made = [m.transpose(1, 2) for m in made]
    rows = sum(fresh)
    mask = None
    if tree_words:
        mask = torch.tensor([r for n in fresh for r in tree_mask(tree(rng, n), tree_words)],
                            dtype=torch.int64).reshape(rows, tree_words)
    return dict(q=(torch.randn((rows, heads, dim), generator=gen) * std).to(dtype), cache_k=made[0], cache_v=made[1],
                table=table, cached=torch.tensor(cached, dtype=torch.int32),
                starts=torch.tensor(np.concatenate([[0], np.cumsum(fresh)]), dtype=torch.int32), mask=mask,
                k_scale=scales[0], v_scale=scales[1], scale=dim ** -0.5)
