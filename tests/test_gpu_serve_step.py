"""The serving example's steps against the definition in 64 bits."""
import importlib.util
import os

import pytest

from tests import attention_cases as C

torch = pytest.importorskip("torch")
from sym_amd import pyreloc as P  # noqa: E402

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "serve_step.py")


def example():
    spec = importlib.util.spec_from_file_location("serve_step", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_steps_over_a_plans_cache():
    ctx = P.Context(0)
    for n, s in enumerate(example().serve(ctx, requests=3, slots=64, steps=3, heads=8, kv_heads=2, dim=64, drafts=5)):
        print("[gpu-case] serve step", n, flush=True)
        torch.cuda.synchronize()
        d = {k: s[k].cpu() for k in ("q", "cache_k", "cache_v", "table", "cached", "k_scale", "v_scale")}
        want, _, bound = C.attention(d["q"], d["cache_k"], d["cache_v"], d["table"], d["cached"], s["tables"].starts.cpu(),
                                     s["tables"].mask.cpu(), 64 ** -0.5, d["k_scale"], d["v_scale"], torch.float16)
        assert bool(((s["out"].double().cpu() - want).abs() <= bound + 2.0 ** -24).all())
        # the rows' slots hold what was appended: each request's, after its context
        page = torch.arange(3)[:, None]
        assert torch.equal(s["tables"].slots.cpu().view(3, 5), page * 64 + d["cached"].long()[:, None] + torch.arange(5))
    ctx.close()
