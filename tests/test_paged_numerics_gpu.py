"""Numbers at the edges of the dense paged operators: weights far below the largest, NaN rows."""

import math

import pytest
import torch

import paged_ref as ref
from paged_ref import D, Cache
from test_paged_attention_gpu import check, layer, queries

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [HF, BF], ids=["fp16", "bf16"])
@pytest.mark.parametrize("G,T", [(1, 1), (4, 3), (4, 8)], ids=["row", "rows12", "rows32"])
@pytest.mark.parametrize("gap,spread", [(12.0, 0.0), (16.0, 1.0), (18.0, 1.0), (17.4, 0.0)])
def test_keys_far_below_a_loud_one_keep_their_share(dtype, G, T, gap, spread):
    """A sink whose score is `gap` nats above all others and whose value is zero: the output is theirs alone.  Enough
    requests over the same pages that a stream lies in one CTA or two.

    The weights of one exponent range are rounded relatively; below 2^-27 of the largest weight fp16 weights are off by
    at most 2^-38 of it each, which the tolerance adds."""
    n, B = 20_000, 200
    one = Cache([n], 1, dtype, 16, "heads", seed=7)
    k, v = one.views()
    g = torch.Generator().manual_seed(11)
    axis = torch.zeros(D)
    axis[3] = 1.0
    rows = 0.25 * torch.randn(n, D, generator=g)
    rows[:, 3] = spread * torch.randn(n, generator=g)  # a query of 1 along the axis: a score of that many nats
    rows[0] = 0.0
    rows[0, 3] = gap + (0.0 if spread == 0 else 4.5)
    vals = 1.0 + 0.25 * torch.randn(n, D, generator=g)
    vals[0] = 0.0
    slot = torch.arange(n, device="cuda")
    t = one.table[0].long()
    k[t[slot // 16], slot % 16, 0], v[t[slot // 16], slot % 16, 0] = rows.to(dtype).cuda(), vals.to(dtype).cuda()
    q = (axis * torch.ones(1, T, G, 1)).to(dtype).cuda()
    o, z, _, tol, ds = ref.attend(one, q, scale=1.0)
    if dtype == HF:
        tol = tol + 2.0**-38 * one.rows(0, 0, n)[1].double().abs().sum(0)
    many = Cache([n], 1, dtype, 16, "heads", seed=7)
    many.kv, many.lens = one.kv, [n] * B
    many.table, many.seq_lens = one.table.expand(B, -1).contiguous(), one.seq_lens.expand(B).contiguous()
    lse = torch.empty(B, T, G, device="cuda")
    out = layer(many, G, T, scale=1.0).forward(q.expand(B, T, G, D).contiguous(), many.seq_lens, lse=lse)
    check(out, lse, tuple(x.expand(B, *x.shape[1:]) if torch.is_tensor(x) else x for x in (o, z, None, tol, ds)))


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T", [1, 3])
def test_a_nan_row_adds_nothing_to_keys_it_does_not_see(dtype, T):
    """One query head of NaN: the weights of the keys it sees become NaN, those of the keys no row sees stay as they are,
    in the tiles that hold both: before the document, outside the window, on a missing page, behind an early token."""
    n, first, window, sinks = 300, 70, 100, 5
    cache = Cache([n, n], 2, dtype, 16, "heads")
    q = queries(cache, 4, T)
    q[0, 0, 1] = math.nan  # the first token of the first request, a head of KV head 0
    cache.table[:, 14] = -1
    mass = torch.rand(2, 2, cache.cap, device="cuda")
    before = mass.clone()
    att = layer(cache, 4, T, window=window, sink_tokens=sinks)
    att.forward(q, cache.seq_lens, first_key=torch.tensor([first, first], dtype=torch.int32, device="cuda"), mass=mass)
    pos = torch.arange(cache.cap, device="cuda")
    there = (pos // 16 != 14) & (pos < n)
    by = [there & ref.visible(pos, n - T + t, first, window, sinks) for t in range(T)]
    for r in range(2):
        for h in range(2):
            nan = by[0] if r == 0 and h == 0 else torch.zeros_like(there)
            seen = torch.stack(by).any(0)
            assert torch.equal(mass[r, h].isnan(), nan), (r, h)
            assert torch.equal(mass[r, h][~seen], before[r, h][~seen]), (r, h)
            assert bool((mass[r, h][seen & ~nan] > before[r, h][seen & ~nan]).all()), (r, h)
