"""Eviction from caches whose block table has entries that name no page: such slots are invisible before and after."""

import math

import pytest
import torch

import paged_ref as ref
from paged_ref import D, Cache
from pqhsa_release_b200 import PagedAttention
from test_paged_attention_gpu import check, layer, queries

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def expected(mass, pos, there, n, budget, sinks, recent, last):
    """Former slot of each of the first min(n, budget) slots: slots that are not there stay below the budget, else go."""
    if n <= budget:
        return list(range(n))

    def key(i):
        if not there[i]:
            return (3, 0.0) if i < budget else (0, 0.0)
        if int(pos[i]) < sinks or int(pos[i]) > last - recent:
            return (2, 0.0)
        x = float(mass[i])
        return (2, 0.0) if x == math.inf else (1, -math.inf if math.isnan(x) else x)

    kept = sorted(sorted(range(n), key=lambda i: tuple(-x for x in key(i)) + (i,))[:budget])
    stay = {i for i in kept if i < budget}
    late = iter([i for i in kept if i >= budget])
    return [i if i in stay else next(late) for i in range(budget)]


GAPS = {
    "behind": lambda blocks, low: [blocks - 1, blocks - 3],  # the sources of kept slots, the most recent among them
    "below": lambda blocks, low: [0, low // 2],              # what would be holes, the sinks' page among them
    "both": lambda blocks, low: list(range(0, blocks, 3)),
    "all_below": lambda blocks, low: list(range(low)),       # no place is left at all
    "all": lambda blocks, low: list(range(blocks)),
}


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("layout,block", [("rows", 16), ("heads", 7), ("heads", 1)])
@pytest.mark.parametrize("gaps", GAPS)
@pytest.mark.parametrize("inplace", [True, False], ids=["inplace", "apart"])
def test_evict_over_a_table_with_gaps(dtype, layout, block, gaps, inplace):
    evict_case(700, 112, 40, 5, 2, dtype, layout, block, gaps, inplace)


@pytest.mark.parametrize("n,budget", [(70_000, 16_384), (400_001, 4096)], ids=["four_ctas", "past_shared_memory"])
def test_evict_long_over_a_table_with_gaps(n, budget):
    evict_case(n, budget, 64, 4, 1, BF, "heads", 64, "both", True)


def evict_case(n, budget, recent, sinks, H, dtype, layout, block, gaps, inplace):
    lens = [n, n // 2, 3]
    cache = Cache(lens, H, dtype, block, layout, seed=3)
    g = torch.Generator().manual_seed(n)
    mass = torch.rand(3, H, cache.cap, generator=g)
    mass[torch.rand(3, H, cache.cap, generator=g) < 0.3] = 0.0
    mass[:, :, 5::50], mass[:, :, 7::90], mass[:, :, 9::70] = math.inf, math.nan, 0.25
    pos = torch.arange(cache.cap, dtype=torch.int32).repeat(3, H, 1)
    blocks, low = -(-n // block), budget // block
    bad = torch.zeros(cache.per, dtype=torch.bool)
    bad[GAPS[gaps](blocks, low)] = True
    names = torch.tensor([-1, cache.kv.shape[1 if layout == "rows" else 0], 2**31 - 1, -(2**31)], dtype=torch.int32)
    cache.table[0] = torch.where(bad, names[torch.arange(cache.per) % 4], cache.table[0].cpu()).cuda()
    there = [~bad[torch.arange(cache.cap) // block], torch.ones(cache.cap, dtype=torch.bool), torch.ones(cache.cap, dtype=torch.bool)]
    att = layer(cache, 2, sink_tokens=sinks)
    kv0 = cache.kv.clone()
    m, p, qp = mass.cuda(), pos.cuda(), cache.seq_lens - 1
    nm, npos = (m, p) if inplace else (torch.full_like(m, 3.0), torch.full_like(p, 3))
    wm, wp = nm.cpu().clone(), npos.cpu().clone()
    source = torch.empty(3, H, budget, dtype=torch.int32, device="cuda")
    new = att.evict(cache.seq_lens.clone(), mass=m, key_pos=p, query_pos=qp, budget=budget, recent=recent, source=source,
                    new_mass=nm, new_pos=npos)
    assert new.tolist() == [min(x, budget) for x in lens]
    want = Cache(lens, H, dtype, block, layout, seed=3)
    want.kv, want.table = kv0, cache.table
    ks, vs = want.views()
    for r, h in ((r, h) for r in range(3) for h in range(H)):
        src = expected(mass[r, h].tolist(), pos[r, h], there[r], lens[r], budget, sinks, recent, lens[r] - 1)
        assert source[r, h].tolist() == src + [-1] * (budget - len(src)), (r, h)
        at = torch.tensor(src, dtype=torch.long)
        wm[r, h, : len(src)], wp[r, h, : len(src)] = mass[r, h][at], pos[r, h][at]
        to = (at != torch.arange(len(src))).nonzero().view(-1)
        fro = at[to]
        assert bool(there[r][to].all()) and bool(there[r][fro].all())  # nothing is moved from or to a page that is missing
        t = want.table[r].long()
        to, fro = to.cuda(), fro.cuda()
        ks[t[to // block], to % block, h] = ks[t[fro // block], fro % block, h].clone()
        vs[t[to // block], to % block, h] = vs[t[fro // block], fro % block, h].clone()
    assert torch.equal(cache.kv, kv0)
    assert torch.equal(nm.cpu().nan_to_num(-3), wm.nan_to_num(-3)) and torch.equal(npos.cpu(), wp)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("missing", [[6, 7], [1], [0, 2, 7]], ids=["late", "early", "mixed"])
def test_append_evict_attend_over_a_table_with_gaps(dtype, missing):
    """Rows appended to missing pages are dropped; after the eviction the attention sees the keys that are there, with
    their own rows and positions, and no other."""
    H, G, block, n, T, budget, recent, sinks = 2, 3, 16, 124, 4, 64, 24, 3
    cache = Cache([n], H, dtype, block, "heads", room=n + T)
    blocks = cache.kv.shape[0]
    true = cache.table.clone()
    cache.table[0, missing] = torch.tensor([-1, blocks, -7][: len(missing)], dtype=torch.int32, device="cuda")
    att = layer(cache, G, T, sink_tokens=sinks)
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(1, T, H, D, generator=g).to(dtype).cuda() for _ in range(2))
    kv0 = cache.kv.clone()
    pos = torch.arange(cache.cap, dtype=torch.int32, device="cuda").repeat(1, H, 1)
    mass = torch.rand(1, H, cache.cap, generator=g).cuda()
    qp = cache.seq_lens - 1 + T
    att.append(k, v, cache.seq_lens, key_pos=pos, query_pos=qp, mass=mass)
    n += T
    # the keys there are, by position, from the pages as they were and the rows appended to pages that are there
    old = Cache([n], H, dtype, block, "heads", room=n)
    old.kv, old.table = kv0.clone(), true
    for t in range(T):
        for h in range(H):
            old.put(0, h, n - T + t, k[0, t, h], v[0, t, h])
    there = torch.tensor([i // block not in missing for i in range(n)])
    m0 = mass[0].cpu().clone()
    att.evict(cache.seq_lens, mass=mass, key_pos=pos, query_pos=qp, budget=budget, recent=recent)
    assert cache.seq_lens.tolist() == [budget]
    q = queries(cache, G, 1)
    out = att.forward(q, cache.seq_lens, key_pos=pos, query_pos=qp)
    # the same keys in a cache of their own, at the same positions
    want = Cache([budget], H, dtype, block, "heads", room=n)
    seen = torch.full((1, H, want.cap), -1, dtype=torch.int32, device="cuda")
    for h in range(H):
        src = expected(m0[h].tolist(), list(range(n)), there.tolist(), n, budget, sinks, recent, n - 1)
        kk, vv = old.rows(0, h, n)
        for i, j in enumerate(src):
            want.put(0, h, i, kk[j], vv[j])
            if there[j]:
                seen[0, h, i] = j
    check(out, None, ref.attend(want, q, sinks=sinks, key_pos=seen, query_pos=[n - 1]))
