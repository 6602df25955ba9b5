"""Serving steps over caches that a relocation plan has laid out.

The C5 plan uploads each request's keys and values, f16 [B, S, heads, dim] on the
host, as int8 [B, heads, S, dim] with a scale a head. That result is a paged
cache as it is: a request's page is its S slots. Each step then drafts a tree of
tokens a request, and three calls take them in:

    block_tables         the drafted tokens' slots, positions and masks
    norm_rotate_append   norms and rotation; keys and values into the cache
    tree_attention       every drafted token attends over the prompt and its
                         own ancestors

after which the accepted tokens, here a chain at the head of the tree, become
part of the context.

    python examples/serve_step.py [--requests 4 --slots 1024 --steps 8]
"""
import argparse
import os
import random
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from sym_amd import attention as A  # noqa: E402
from sym_amd import pyreloc as P  # noqa: E402
from sym_amd import workloads as W  # noqa: E402

CHAIN = 2  # drafted tokens that a step accepts: the tree's first two


def upload(ctx, requests, slots, heads, dim, seed):
    """The plan's result on the GPU, [requests, heads, slots, dim], and its scales."""
    x, scale = W.c5_input(requests, slots, heads, dim, seed)
    bound = P.Bound(P.Plan(W.c5_plan(heads, dim).blob), {"B": requests, "S": slots}, W.param("scale", scale))
    out = torch.empty((requests, heads, slots, dim), dtype=torch.int8, device="cuda:%d" % ctx.device)
    ctx.execute_h2d(bound, x.ctypes.data, x.nbytes, out.data_ptr(), out.numel())
    return out, torch.from_numpy(scale).to(out.device)


def serve(ctx, requests=4, slots=1024, steps=8, heads=32, kv_heads=8, dim=128, drafts=12, seed=0):
    """Yields, after each step, what went into it and what came out."""
    device = torch.device("cuda:%d" % ctx.device)
    rng, gen = random.Random(seed), torch.Generator(device=device).manual_seed(seed)
    (keys, k_scale), (values, v_scale) = (upload(ctx, requests, slots, kv_heads, dim, seed + i) for i in range(2))
    cache_k, cache_v = keys.transpose(1, 2), values.transpose(1, 2)  # [pages, page, kv_heads, dim]
    i32 = dict(dtype=torch.int32, device=device)
    most = slots - steps * CHAIN - drafts
    if most < 1:
        raise ValueError("%d slots are too few for %d steps" % (slots, steps))
    cached = torch.tensor([rng.randint(1, most) for _ in range(requests)], **i32)
    fresh = torch.full((requests,), drafts, **i32)
    table = torch.arange(requests, **i32)[:, None]
    no_pages = torch.empty(0, **i32)  # every request has its page already
    half = torch.arange(dim // 2, device=device) / (dim // 2)
    angle = torch.arange(slots, device=device)[:, None] * 10000.0 ** -half
    cos, sin = angle.cos(), angle.sin()
    weights = [torch.rand(dim, generator=gen, device=device).to(torch.float16) for _ in range(2)]
    rows = requests * drafts
    room = torch.empty(A.tree_attention_workspace(rows, requests, heads, kv_heads, dim, slots), dtype=torch.uint8,
                       device=device)
    for _ in range(steps):
        # a token follows the one before or an earlier one; the first two are a chain
        parents = torch.tensor([-1 if j == 0 else 0 if j == 1 else rng.randrange(j) for _ in range(requests)
                                for j in range(drafts)], **i32)
        # stands for the projections of the step's hidden states
        fused = torch.randn((rows, heads + 2 * kv_heads, dim), generator=gen, device=device).to(torch.float16)
        q, k, v = fused.split((heads, kv_heads, kv_heads), 1)
        t = A.block_tables(ctx, cached, fresh, table, no_pages, slots, rows, parents=parents)
        turned = A.norm_rotate_append(ctx, q, k, v, t.slots, cache_k, cache_v, t.positions, cos, sin, *weights, 1e-6,
                                      k_scale=k_scale, v_scale=v_scale)
        out = A.tree_attention(ctx, turned, cache_k, cache_v, table, cached, t.starts, mask=t.mask, k_scale=k_scale,
                               v_scale=v_scale, workspace=room)
        yield dict(q=turned, cache_k=cache_k, cache_v=cache_v, table=table, cached=cached, tables=t, k_scale=k_scale,
                   v_scale=v_scale, out=out)
        cached = cached + CHAIN


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--requests", type=int, default=4)
    p.add_argument("--slots", type=int, default=1024)
    p.add_argument("--steps", type=int, default=8)
    a = p.parse_args()
    ctx = P.Context(0)
    for n, s in enumerate(serve(ctx, a.requests, a.slots, a.steps)):
        print("step %d: contexts of %s tokens, result %s, root mean square %.4f"
              % (n, s["cached"].tolist(), list(s["out"].shape), float(s["out"].float().square().mean().sqrt())))
    torch.cuda.synchronize()
    ctx.close()


if __name__ == "__main__":
    main()
