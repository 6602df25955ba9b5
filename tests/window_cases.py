"""Plain 64-bit forms of attention with a window and first tokens that stay, of
caches with a scale a block, and inputs for them."""
import random

import torch

from tests import attention_cases as C

F32, ROUND = C.F32, C.ROUND
# f16 numbers below 2^-14 lie 2^-24 apart: a result's rounding there is off by half of that
STEP = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
LEAST = 2.0 ** -126
MANY = 1 << 40


# ------------------------------------------------------------ blocks of a cache

def block_append(k, v, cache_k, cache_v, k_scale, v_scale, table, cached, starts):
    """Token by token, in the 32-bit steps of the definition (exact: no other result
    is right). Returns new caches and scales."""
    out = []
    for new, cache, scale in ((k, cache_k, k_scale), (v, cache_v, v_scale)):
        cache, scale = cache.clone(), scale.clone()
        pages, page = cache.shape[:2]
        block = page // scale.shape[1]
        for b in range(table.shape[0]):
            have, x = int(cached[b]), int(cached[b])
            end = min(have + int(starts[b + 1] - starts[b]), table.shape[1] * page)
            while x < end:
                first = x - x % block
                stop = min(first + block, end)
                at, off = int(table[b, first // page]), first % page
                rows = new[int(starts[b]) + x - have:int(starts[b]) + stop - have].float()
                if 0 <= at < pages:
                    most = torch.where(rows.isfinite(), rows.abs(), 0.0).amax((0, 2))
                    old = scale[at, off // block].clone()
                    now = (most * torch.tensor(1.0 / 127.0, dtype=torch.float32)).clamp(min=LEAST)
                    if x > first:
                        now = torch.maximum(now, old)
                        kept = cache[at, off:off + x - first].float() * (old * (1.0 / now))[:, None]
                        cache[at, off:off + x - first] = kept.round().clamp(-128, 127).to(torch.int8)
                    y = rows * (1.0 / now)[:, None]
                    y = torch.where(y.isnan(), -128.0, y).clamp(-128, 127).round()
                    cache[at, off + x - first:off + stop - first] = y.to(torch.int8)
                    scale[at, off // block] = now
                x = stop
        out += [cache, scale]
    return out[0], out[2], out[1], out[3]


def values(codes, scale, dtype=torch.float64):
    block = codes.shape[1] // scale.shape[1]
    return codes.to(dtype) * scale.to(dtype).repeat_interleave(block, 1)[..., None]


# ------------------------------------------------------------ attention over a cache

def view_attention(q, keys, vals, table, cached, starts, mask, scale, k_scale, v_scale, window, sinks, round_to):
    """(result, lse, error bound), row by row in 64 bits on the CPU."""
    rows, heads, dim = q.shape
    pages, page, kv, _ = keys.shape
    out = torch.zeros((rows, heads, dim), dtype=torch.float64)
    bound = torch.zeros_like(out)
    lse = torch.full((rows, heads), -float("inf"), dtype=torch.float64)
    group, columns, u = heads // kv, table.shape[1], ROUND[round_to]
    most_scale = None
    if k_scale is not None:
        if k_scale.dim() == 1:
            k_scale, v_scale = (z[None, None].expand(pages, 1, kv) for z in (k_scale, v_scale))
        keys, vals = values(keys, k_scale), values(vals, v_scale)
        most_scale = float(v_scale.abs().max())
    window, sinks = min(window or MANY, MANY), min(sinks, MANY)
    for b in range(table.shape[0]):
        r0, r1 = int(starts[b]), int(starts[b + 1])
        if r1 <= r0:
            continue
        c = int(cached[b])
        limit = min(c + r1 - r0, columns * page)
        ids = table[b].long().repeat_interleave(page)[:limit]
        x = torch.arange(limit)
        there = (ids >= 0) & (ids < pages)
        k = keys[ids.clamp(0, pages - 1), x % page].double()
        v = vals[ids.clamp(0, pages - 1), x % page].double()
        rows_of = None if mask is None else mask[r0:r1].tolist()
        see = C.visible(c, r1 - r0, limit, rows_of) & there[None, :]
        for j in range(r1 - r0):
            depth = j if rows_of is None else max(0, sum(bin(w & (2 ** 64 - 1)).count("1") for w in rows_of[j]) - 1)
            near = (x < sinks) | (c + depth - x < window)
            if mask is not None:
                near |= x >= c
            see[j] &= near
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
                # scores in 32 bits (products, their sum, two scales): their error is the weights'
                # relative one; weights are rounded to the result's type (f16: to 2^-31 of the sum
                # at least, of scaled values to 2^-30 of the largest), the sums and the result once more
                ds = (dim + 6) * F32 * float((kk.abs() @ q[r0 + j, h].double().abs()).max()) * abs(scale)
                size = p @ vv.abs()
                steps = at.numel() / 32 + 16
                least = vv.abs().amax(0) * 2.0 ** -31 if most_scale is None else most_scale * 128 * 2.0 ** -30
                bound[r0 + j, h] = u * o.abs() + STEP[round_to] + (u + 2 * ds + (steps + 2) * F32) * size + at.numel() * least
    return out, lse, bound


def view_case(seed, cached, fresh, heads, kv, dim, dtype, cache, page, block=None, order="slots", tree_words=0, columns=None,
              std=1.0):
    """Operands on the CPU; `block`: an int8 cache with a scale a block."""
    s = C.attention_case(seed, cached, fresh, heads, kv, dim, dtype, cache, page, order, tree_words, columns, std)
    if block:
        gen = torch.Generator().manual_seed(seed + 1)
        shape = (s["cache_k"].shape[0], page // block, kv)
        s["k_scale"], s["v_scale"] = (torch.exp(torch.randn(shape, generator=gen)) * 0.01 for _ in range(2))
    return s


# ------------------------------------------------------------ packed sequences

def sees(n, window, sinks):
    p = torch.arange(n)
    back = p[:, None] - p[None, :]
    return (back >= 0) & ((p[None, :] < sinks) | (back < (window or MANY)))


def window_attention(q, k, v, starts, window, sinks, scale, dout=None, round_to=None):
    """Results in 64 bits, and bounds of a kernel's errors: of the result, the
    logarithm of the sum, and with `dout` the gradients dq, dk, dv.

    A kernel's scores are 32-bit sums of exact products: off by ds, which is the
    weights' relative error. Weights P are rounded to `round_to` for a product, and
    so are dS = P (dP - D) scale: each u relative, or 2^-24 of the largest it may
    be where f16 ends (both are scaled to be near it). D is of the rounded result."""
    rows, heads, dim = q.shape
    half = round_to or q.dtype
    group, u = heads // k.shape[1], ROUND[half]
    q, k, v = q.double(), k.double(), v.double()
    o, lse = torch.zeros_like(q), torch.full((heads, rows), -float("inf"), dtype=torch.float64)
    bo = torch.zeros_like(o)
    out = dict(o=o, lse=lse, bo=bo, ds=torch.zeros(heads, rows, dtype=torch.float64))
    if dout is not None:
        dout = dout.double()
        for name, like in (("dq", q), ("dk", k), ("dv", v)):
            out[name], out["b" + name] = torch.zeros_like(like), torch.zeros_like(like)
    for a, b in zip(starts.tolist(), starts.tolist()[1:]):
        if b <= a:
            continue
        see = sees(b - a, window, sinks)
        for h in range(heads):
            qq, kk, vv = q[a:b, h], k[a:b, h // group], v[a:b, h // group]
            s = torch.where(see, qq @ kk.T * scale, -float("inf"))
            p = torch.softmax(s, 1)
            o[a:b, h] = p @ vv
            lse[h, a:b] = torch.logsumexp(s, 1)
            # of a row: of its largest score
            ds = (dim + 4) * F32 * torch.where(see, qq.abs() @ kk.abs().T, 0.0).amax(1) * abs(scale) + 4 * F32 * s.masked_fill(~see, 0.0).abs().amax(1)
            out["ds"][h, a:b] = ds
            steps = (b - a) / 32 + 16
            rel = u + 2 * ds[:, None] + steps * F32
            least = 2.0 ** -30  # of weights that are at most one
            bo[a:b, h] = u * o[a:b, h].abs() + STEP[half] + rel * (p @ vv.abs()) + least * (see.double() @ vv.abs())
            if dout is None:
                continue
            do = dout[a:b, h]
            dp = do @ vv.T
            size_p = do.abs() @ vv.abs().T
            d = (do * o[a:b, h]).sum(1, keepdim=True)
            size_d = (do.abs() * (o[a:b, h].abs() * (u + dim * F32) + bo[a:b, h])).sum(1, keepdim=True)
            g = p * (dp - d) * scale
            # dP and D in 32 bits, D of the rounded result
            off = p * abs(scale) * ((u + 2 * ds[:, None] + 8 * F32) * (dp - d).abs() + (dim + 4) * F32 * size_p + size_d)
            off = off + see * least * abs(scale) * float(do.abs().max()) * float(vv.abs().max()) * dim
            out["dq"][a:b, h] += g @ kk
            out["dk"][a:b, h // group] += g.T @ qq
            out["dv"][a:b, h // group] += p.T @ do
            sums = steps * group * F32
            out["bdq"][a:b, h] += (off + sums * g.abs()) @ kk.abs()
            out["bdk"][a:b, h // group] += (off + sums * g.abs()).T @ qq.abs()
            out["bdv"][a:b, h // group] += ((u + 2 * ds[:, None] + sums) * p + see * least).T @ do.abs()
    if dout is not None:
        for name in ("dq", "dk", "dv"):
            out["b" + name] += u * out[name].abs() + STEP[half]
    return out


def window_case(seed, lengths, heads, kv, dim, dtype, before=0, after=0, fused=True, std=1.0):
    """Packed sequences on the CPU, with rows of no sequence `before` and `after` them."""
    gen = torch.Generator().manual_seed(seed)
    rows = before + sum(lengths) + after
    whole = (torch.randn((rows, heads + 2 * kv, dim), generator=gen) * std).to(dtype)
    q, k, v = whole.split((heads, kv, kv), 1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    starts = [before]
    for n in lengths:
        starts.append(starts[-1] + n)
    return dict(q=q, k=k, v=v, starts=torch.tensor(starts, dtype=torch.int32),
                dout=(torch.randn((rows, heads, dim), generator=gen) * std).to(dtype))


def ragged(seed, n, longest):
    rng = random.Random(seed)
    return [rng.randint(0, longest) for _ in range(n)]
