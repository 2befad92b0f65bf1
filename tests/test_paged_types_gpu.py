"""The dense paged operators' cases in the types that the other files do not run them in."""

import math

import pytest
import torch

from paged_ref import D, Cache
from pqhsa_release_b200 import EvictingCacheAdapter
from test_evicting_cache_gpu import simulate
from test_paged_attention_gpu import evict_case

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("layout,block", [("rows", 16), ("heads", 7)])
@pytest.mark.parametrize("inplace", [True, False], ids=["inplace", "apart"])
@pytest.mark.parametrize("budget,recent,sinks", [(64, 10, 4), (1, 0, 0), (500, 100, 0)])
def test_evict_fp16(layout, block, inplace, budget, recent, sinks):
    lens = [700, 64, 0, 1, 501, -3]
    g = torch.Generator().manual_seed(budget)
    cap = Cache(lens, 2, HF, block, layout).cap
    mass = torch.rand(6, 2, cap, generator=g)
    mass[torch.rand(6, 2, cap, generator=g) < 0.3] = 0.0
    mass[0, 1, 3], mass[0, 1, 5], mass[0, 1, 9] = math.nan, -0.0, math.inf
    pos = torch.arange(cap, dtype=torch.int32).repeat(6, 2, 1)
    pos[4, 1, :501] = torch.randperm(501, generator=g).int()
    evict_case(lens, 2, HF, block, layout, budget, recent, sinks, mass.cuda(), pos.cuda(), [n - 1 for n in lens], inplace)


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("S,with_queries", [(300, True), (300, False), (40, False), (100, True)])
def test_adapter_follows_the_rule_in_16_bits(dtype, S, with_queries):
    """The rule in 64 bits over the same 16-bit numbers: which keys stay goes by fp32 weights, so it is the same.

    An output is off by half a step of its own, by half a step of every weight (p is rounded for the product with the
    values: half a step times the sum of w |v|, which the rule over |v| gives), and by the scores' rounding as in fp32:
    2^-23 (2 x 130 x 60 + 400) of that sum."""
    B, H, G, budget, interval, sinks, recent, steps = 2, 2, 4, 64, 16, 3, 20, 40
    g = torch.Generator().manual_seed(S + 1)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)
    keys, values = r(B, H, S, D), r(B, H, S, D)
    wq = r(B, H * G, 13, D) if with_queries else None
    toks = [(r(B, H * G, D), r(B, H, D), r(B, H, D)) for _ in range(steps)]
    qs = [t[0] for t in toks]
    want, kept, mass = simulate(keys, values, qs, toks, budget, interval, sinks, recent, wq)
    size, _, _ = simulate(keys, values.abs(), qs, [(q, k, v.abs()) for q, k, v in toks], budget, interval, sinks, recent, wq)
    ad = EvictingCacheAdapter(num_query_heads=H * G, num_kv_heads=H, budget=budget, interval=interval, sink_tokens=sinks, recent=recent)
    ad.build_cache(keys.cuda(), values.cuda(), None if wq is None else wq.cuda())
    half = torch.finfo(dtype).eps / 2
    for i, (q, k, v) in enumerate(toks):
        ctx = ad.decode_step(q.cuda(), k.cuda(), v.cuda()).context.double().cpu()
        assert ((ctx - want[i]).abs() <= half * want[i].abs() + (half + 2.0**-23 * (2 * 130 * 60 + 400)) * size[i] + 2.0**-24).all(), i
    assert (ad.evictions > 0) == (S + steps > budget + interval)  # 40 + 40 tokens just fill it
    for b in range(B):
        for h in range(H):
            assert ad.positions[b, h, : ad.length].tolist() == kept[b][h]
            assert (ad.weights[b, h, : ad.length].double().cpu() - mass[b][h]).abs().max() <= 1e-3
