"""Calls of the evicting adapter at its edges: odd inputs, refusals that must change nothing, captures."""

import pytest
import torch

from paged_ref import D
from pqhsa_release_b200 import EvictingCacheAdapter

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def rows(*shape, dtype=BF, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def state(ad):
    """Everything an adapter is, its device tensors copied."""
    return ((ad.length, ad.position, ad.evictions, id(ad.attention)),
            [t.clone() for t in (ad.keys, ad.values, ad.positions, ad.weights, ad.lens, ad.query_pos)])


def same(a, b):
    return a[0] == b[0] and all(torch.equal(x, y) for x, y in zip(a[1], b[1]))


def filled(dtype=BF, tokens=40, **kw):
    """An adapter of two requests whose next append evicts."""
    ad = EvictingCacheAdapter(num_query_heads=8, num_kv_heads=2, budget=32, interval=8, sink_tokens=2, recent=4, **kw)
    k, v = rows(2, 2, tokens, D, dtype=dtype, seed=1), rows(2, 2, tokens, D, dtype=dtype, seed=2)
    ad.build_cache(k[:, :, : tokens - 1], v[:, :, : tokens - 1])
    ad.append(k[:, :, tokens - 1], v[:, :, tokens - 1])
    return ad


def shifted(x):
    """The same values one element off a 16-byte boundary, contiguous."""
    odd = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape)
    return odd.copy_(x)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
def test_rows_off_a_16_byte_boundary(dtype):
    a, b = filled(dtype), filled(dtype)
    for i in range(12):
        k, v, q = rows(2, 2, D, dtype=dtype, seed=10 + i), rows(2, 2, D, dtype=dtype, seed=30 + i), rows(2, 8, D, dtype=dtype, seed=50 + i)
        want = a.decode_step(q, k, v).context
        assert torch.equal(b.decode_step(q, shifted(k), shifted(v) if i % 2 else v).context, want), i
    sa, sb = state(a), state(b)
    assert sa[0][:3] == sb[0][:3] == (36, 52, 2) and all(torch.equal(x, y) for x, y in zip(sa[1], sb[1]))


def test_a_step_with_bad_queries_appends_nothing():
    ad = filled()
    before = state(ad)
    k, v, q = rows(2, 2, D, seed=3), rows(2, 2, D, seed=4), rows(2, 8, D, seed=5)
    for bad in (q[:1], q[:, :4], q[:, :, :64], q.float(), q.cpu(), q[0], q.to(HF)):
        with pytest.raises(ValueError, match="queries"):
            ad.decode_step(bad, k, v)
        assert same(state(ad), before), tuple(bad.shape)
    assert ad.decode_step(q, k, v).context.shape == q.shape and ad.position == 41
    with pytest.raises(RuntimeError, match="build_cache"):
        EvictingCacheAdapter(num_query_heads=8, num_kv_heads=2, budget=32, recent=4).decode_step(q, k, v)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
def test_queries_in_any_strides(dtype):
    ad = filled(dtype)
    q = rows(2, 8, D, dtype=dtype, seed=5)
    want = ad.forward(q).context
    wide = torch.empty(2, 9, 2 * D, dtype=dtype, device="cuda")
    forms = [wide[:, 1:, :D], wide[:, :8, 4 : 4 + D], wide[:, :8, ::2], torch.empty(8, 2, D, dtype=dtype, device="cuda").transpose(0, 1),
             torch.empty(2, D, 8, dtype=dtype, device="cuda").transpose(1, 2), torch.empty(2 * 8 * D + 1, dtype=dtype, device="cuda")[1:].view(2, 8, D)]
    for f in forms:
        f.copy_(q)
        assert torch.equal(ad.forward(f).context, want), f.stride()


@pytest.mark.parametrize("why", ["queries_elsewhere", "values_shape", "queries_dtype", "group", "dtype"])
def test_a_refused_prompt_leaves_the_cache_there_was(why):
    ad = filled()
    before = state(ad)
    k, wq = rows(2, 2, 60, D, seed=8), rows(2, 8, 5, D, seed=9)
    values, queries = k, wq
    if why == "queries_elsewhere":
        queries = wq.cpu()
    elif why == "values_shape":
        values = k[:, :, :-1]
    elif why == "queries_dtype":
        queries = wq.float()
    elif why == "dtype":
        k = values = k.double()
        queries = wq.double()
    if why == "group":  # 32 query heads per KV head: more than a layer takes
        ad = EvictingCacheAdapter(num_query_heads=64, num_kv_heads=2, budget=32, interval=8, recent=4)
        with pytest.raises(ValueError, match="query heads per KV head"):
            ad.build_cache(k, values)
        with pytest.raises(RuntimeError, match="build_cache"):
            ad.append(k[:, :, 0], k[:, :, 0])
        return
    with pytest.raises(ValueError):
        ad.build_cache(k, values, queries)
    assert same(state(ad), before)
    q = rows(2, 8, D, seed=5)
    twin = filled()
    twin.append(rows(2, 2, D, seed=3), rows(2, 2, D, seed=4))
    ad.append(rows(2, 2, D, seed=3), rows(2, 2, D, seed=4))
    assert torch.equal(ad.forward(q).context, twin.forward(q).context)


def test_a_prompts_queries_in_any_strides():
    k, v, wq = rows(2, 2, 60, D, seed=8), rows(2, 2, 60, D, seed=6), rows(2, 8, 13, D, seed=9)
    a = EvictingCacheAdapter(num_query_heads=8, num_kv_heads=2, budget=32, interval=8, sink_tokens=2, recent=4).build_cache(k, v, wq)
    odd = shifted(wq)
    wide = torch.empty(2, 13, 8, D + 4, dtype=BF, device="cuda")[..., 4:].transpose(1, 2)
    wide.copy_(wq)
    for q in (odd, wide, wq.transpose(1, 2).contiguous().transpose(1, 2)):
        b = EvictingCacheAdapter(num_query_heads=8, num_kv_heads=2, budget=32, interval=8, sink_tokens=2, recent=4).build_cache(k, v, q)
        assert all(torch.equal(x, y) for x, y in zip(state(a)[1], state(b)[1]))


def test_what_counts_on_the_host_is_not_captured():
    """Replays of a captured append would go past the room without an eviction, and their rows would be dropped."""
    ad = filled()
    ad.append(rows(2, 2, D, seed=3), rows(2, 2, D, seed=4))
    before = state(ad)
    k, v, q = rows(2, 2, D, seed=13), rows(2, 2, D, seed=14), rows(2, 8, D, seed=5)
    calls = {"append": lambda: ad.append(k, v), "decode": lambda: ad.decode_step(q, k, v), "build": lambda: ad.build_cache(k[:, :, None], v[:, :, None])}
    for name, call in calls.items():
        one, g = torch.zeros(1, device="cuda"), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            one.add_(1.0)  # the capture itself goes on
            with pytest.raises(RuntimeError, match="captured"):
                call()
        g.replay()
        torch.cuda.synchronize()
        assert one.item() == 1.0 and same(state(ad), before), name
    # the attention alone: each replay accumulates its weights, as an eager call does
    twin = filled()
    twin.append(rows(2, 2, D, seed=3), rows(2, 2, D, seed=4))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ad.forward(q).context
    for _ in range(3):
        g.replay()
        want = twin.forward(q).context
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(ad.weights, twin.weights)
    ad.append(k, v)
    twin.append(k, v)
    g.replay()
    want = twin.forward(q).context
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(ad.weights, twin.weights)
