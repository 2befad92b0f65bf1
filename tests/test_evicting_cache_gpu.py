"""Append, attention, weights and eviction together as a user runs them: the evicting adapter over many steps against a
64-bit simulation, a captured step loop, and the vLLM hook's dense steps."""

import math
from types import SimpleNamespace as NS

import pytest
import torch

import paged_ref as ref
from paged_ref import D, Cache
from pqhsa_release_b200 import EvictingCacheAdapter, PagedAttention

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def simulate(keys, values, queries, steps, budget, interval, sinks, recent, window_q=None):
    """The adapter's rule in 64 bits on the host: per head a list of kept tokens; yields the contexts of every step."""
    B, H, S, _ = keys.shape
    G = queries[0].shape[1] // H
    scale = 1 / math.sqrt(D)
    kept = [[list(range(S)) for _ in range(H)] for _ in range(B)]
    mass = [[torch.zeros(S, dtype=torch.float64) for _ in range(H)] for _ in range(B)]

    def weights(b, h, q):  # q [G, D] sees all kept tokens
        s = scale * (q.double() @ keys_all[b][h][kept[b][h]].T)
        return torch.softmax(s, 1)

    def drop(b, h, last):
        toks, m = kept[b][h], mass[b][h]
        src = ref.evict(m.tolist(), toks, len(toks), budget, sinks, recent, last)
        kept[b][h], mass[b][h] = [toks[i] for i in src], m[src]

    keys_all = [[keys[b, h].double() for h in range(H)] for b in range(B)]
    vals_all = [[values[b, h].double() for h in range(H)] for b in range(B)]
    if window_q is not None:
        W = window_q.shape[2]
        for b in range(B):
            for h in range(H):
                for w in range(W):
                    n = S - W + w + 1
                    s = scale * (window_q[b, h * G : (h + 1) * G, w].double() @ keys_all[b][h][:n].T)
                    mass[b][h][:n] += torch.softmax(s, 1).sum(0)
    n = S
    if n >= budget + interval:
        for b in range(B):
            for h in range(H):
                drop(b, h, S - 1)
        n = budget
    out = []
    for i, (q, k, v) in enumerate(steps):
        pos = S + i
        if n >= budget + interval:
            for b in range(B):
                for h in range(H):
                    drop(b, h, pos - 1)
            n = budget
        ctx = torch.zeros(B, H * G, D, dtype=torch.float64)
        for b in range(B):
            for h in range(H):
                keys_all[b][h] = torch.cat([keys_all[b][h], k[b, h].double()[None]])
                vals_all[b][h] = torch.cat([vals_all[b][h], v[b, h].double()[None]])
                kept[b][h].append(pos)
                mass[b][h] = torch.cat([mass[b][h], torch.zeros(1, dtype=torch.float64)])
                w = weights(b, h, q[b, h * G : (h + 1) * G])
                ctx[b, h * G : (h + 1) * G] = w @ vals_all[b][h][kept[b][h]]
                mass[b][h] += w.sum(0)
        n += 1
        out.append(ctx)
    return out, kept, mass


@pytest.mark.parametrize("S,with_queries", [(300, True), (300, False), (40, False), (100, True), (64 + 16, True)])
def test_adapter_follows_the_rule_over_many_steps(S, with_queries):
    B, H, G, budget, interval, sinks, recent, steps = 2, 2, 4, 64, 16, 3, 20, 60
    g = torch.Generator().manual_seed(S)
    r = lambda *s: torch.randn(*s, generator=g)
    keys, values = r(B, H, S, D), r(B, H, S, D)
    wq = r(B, H * G, 13, D) if with_queries else None
    toks = [(r(B, H * G, D), r(B, H, D), r(B, H, D)) for _ in range(steps)]
    want, kept, mass = simulate(keys, values, [t[0] for t in toks], toks, budget, interval, sinks, recent, wq)
    ad = EvictingCacheAdapter(num_query_heads=H * G, num_kv_heads=H, budget=budget, interval=interval, sink_tokens=sinks, recent=recent)
    kc, vc = keys.cuda(), values.cuda()
    ad.build_cache(kc, vc, None if wq is None else wq.cuda())
    assert torch.equal(kc.cpu(), keys) and torch.equal(vc.cpu(), values)
    for i, (q, k, v) in enumerate(toks):
        ctx = ad.decode_step(q.cuda(), k.cuda(), v.cuda()).context.double().cpu()
        # fp32: a score off by 130 roundings of sum|qk| <= 60, weights by twice that, at most 80 + 300 additions
        assert (ctx - want[i]).abs().max() <= 2.0**-23 * (2 * 130 * 60 + 400) * 4, i
        assert ad.length <= budget + interval and ad.position == S + i + 1
    assert ad.lens.tolist() == [ad.length] * B and ad.evictions >= 2
    for b in range(B):
        for h in range(H):
            assert ad.positions[b, h, : ad.length].tolist() == kept[b][h]
            assert (ad.weights[b, h, : ad.length].double().cpu() - mass[b][h]).abs().max() <= 1e-3


def test_adapter_refusals():
    with pytest.raises(ValueError, match="GQA"):
        EvictingCacheAdapter(num_query_heads=5, num_kv_heads=2, budget=8)
    with pytest.raises(ValueError, match="budget"):
        EvictingCacheAdapter(num_query_heads=4, num_kv_heads=2, budget=8, recent=6, sink_tokens=4)
    ad = EvictingCacheAdapter(num_query_heads=4, num_kv_heads=2, budget=8, recent=2, sink_tokens=1)
    x = torch.zeros(1, 2, D, device="cuda")
    with pytest.raises(RuntimeError, match="build_cache"):
        ad.append(x, x)
    with pytest.raises(RuntimeError, match="build_cache"):
        ad.forward(x)
    with pytest.raises(ValueError, match="keys and values"):
        ad.build_cache(x[:, :, None], x)
    ad.build_cache(x[:, :, None], x[:, :, None])
    with pytest.raises(ValueError, match="queries"):
        ad.forward(x)
    with pytest.raises(ValueError, match="keys and values"):
        ad.append(x[:, :1], x[:, :1])
    with pytest.raises(ValueError, match="required"):
        ad.decode_step(torch.zeros(1, 4, D, device="cuda"))


def test_captured_loop_of_append_attention_and_eviction():
    """One graph of a step with all three operators, replayed: the device-side lengths carry it from step to step."""
    B, H, G, budget = 2, 2, 2, 48
    cache = Cache([48, 30], H, BF, 16, "heads", room=80)
    att = PagedAttention(num_query_heads=H * G, num_kv_heads=H, max_requests=B, token_capacity=cache.cap, dtype=BF, device="cuda", sink_tokens=2)
    att.bind_kv_paged(cache.kv, cache.table)
    twin = Cache([48, 30], H, BF, 16, "heads", room=80)

    def state(c):
        return (c.seq_lens, torch.arange(c.cap, dtype=torch.int32, device="cuda").repeat(B, H, 1),
                torch.tensor([47, 29], dtype=torch.int32, device="cuda"), torch.rand(B, H, c.cap, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda"))

    q = torch.empty(B, H * G, D, dtype=BF, device="cuda")
    k, v, out = torch.empty(B, H, D, dtype=BF, device="cuda"), torch.empty(B, H, D, dtype=BF, device="cuda"), torch.empty_like(q)

    def step(a, s):
        lens, pos, qp, mass = s
        qp.add_(1)
        a.append(k, v, lens, key_pos=pos, query_pos=qp, mass=mass)
        a.forward(q, lens, out=out, key_pos=pos, query_pos=qp, mass=mass)
        a.evict(lens, mass=mass, key_pos=pos, query_pos=qp, budget=budget, recent=8)

    eager = PagedAttention(num_query_heads=H * G, num_kv_heads=H, max_requests=B, token_capacity=cache.cap, dtype=BF, device="cuda", sink_tokens=2)
    eager.bind_kv_paged(twin.kv, twin.table)
    s1, s2 = state(cache), state(twin)
    saved = [t.clone() for t in s1]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(att, s1)
    for t, x in zip(s1, saved):
        t.copy_(x)
    gen = torch.Generator(device="cuda").manual_seed(9)
    for i in range(30):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
        graph.replay()
        got = out.clone()
        step(eager, s2)
        torch.cuda.synchronize()
        assert torch.equal(got, out), i
        assert s1[0].tolist() == [budget, min(30 + i + 1, budget)]
    for a, b in zip((*s1, cache.kv), (*s2, twin.kv)):
        assert torch.equal(a, b)


# ---- the vLLM hook ------------------------------------------------------------------------------------------


def metadata(cache, T=1, **kw):
    lens = cache.seq_lens
    slots = []
    for r, n in enumerate(cache.lens):
        for p in range(n - T, n):
            slots.append(int(cache.table[r, p // cache.block]) * cache.block + p % cache.block)
    return NS(use_cascade=False, max_query_len=T, num_actual_tokens=len(cache.lens) * T, seq_lens=lens, seq_lens_cpu=lens.cpu(),
              max_seq_len=max(cache.lens), block_table=cache.table, slot_mapping=torch.tensor(slots, device="cuda"), **kw)


@pytest.mark.parametrize("layout", ["rows", "heads"])
@pytest.mark.parametrize("T", [1, 3])
def test_hook_serves_short_requests_with_the_dense_kernel(layout, T, monkeypatch):
    from pqhsa_release_b200.pq_hsa_vllm import runtime

    for k, v in {"PQ_HSA_BATCH": "1", "PQ_HSA_ENABLE": "1", "PQ_HSA_DENSE": "1", "PQ_HSA_MULTI_QUERY": "0"}.items():
        monkeypatch.setenv(k, v)
    runtime.reset()
    H, G = 2, 4
    cache = Cache([70, 5, 131], H, BF, 16, layout)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(3 * T, H * G, D, generator=g).to(BF).cuda()
    # the step's rows: already in the pages with the newer layout, stored by the hook with the older one
    k, v = torch.randn(2, 3 * T, H, D, generator=g).to(BF).cuda()
    for r, n in enumerate(cache.lens):
        for t in range(T):
            for h in range(H):
                cache.put(r, h, n - T + t, k[r * T + t, h], v[r * T + t, h])
    filled = cache.kv.clone()
    if layout == "rows":
        for r, n in enumerate(cache.lens):
            for t in range(T):
                cache.put(r, slice(None), n - T + t, torch.zeros(D, dtype=BF), torch.zeros(D, dtype=BF))
    impl = NS(scale=0.1, num_heads=H * G, num_kv_heads=H, sliding_window=(39, 0), logits_soft_cap=15.0, alibi_slopes=None)
    layer, out = object(), torch.zeros_like(q)
    calls = []

    def original(impl_, layer_, *a, output=None, **kw):
        calls.append(1)
        return output

    md = metadata(cache, T)
    assert runtime.pq_or_dense_forward(original, impl, layer, q, k, v, cache.kv, md, output=out) is out
    assert not calls and runtime.STATS["library_dense_steps"] == 1 and runtime.STATS["dense_steps"] == 0
    assert torch.equal(cache.kv, filled)
    o, _, _, tol, _ = ref.attend(cache, q.view(3, T, H * G, D), scale=0.1, softcap=15.0, window=40)
    assert ((out.view(3, T, H * G, D).double() - o).abs() <= tol).all()
    # off by default, and a prefill step is the original's in any case
    monkeypatch.setenv("PQ_HSA_DENSE", "0")
    runtime.pq_or_dense_forward(original, impl, layer, q, k, v, cache.kv, md, output=out)
    monkeypatch.setenv("PQ_HSA_DENSE", "1")
    md2 = metadata(cache, T)
    md2.max_query_len, md2.num_actual_tokens = 64, 192
    runtime.pq_or_dense_forward(original, impl, layer, q, k, v, cache.kv, md2, output=out)
    assert len(calls) == 2 and runtime.STATS["dense_steps"] == 2
    runtime.reset()


def test_a_refused_append_changes_nothing():
    from pqhsa_release_b200 import EvictingCacheAdapter

    ad = EvictingCacheAdapter(num_query_heads=8, num_kv_heads=2, budget=32, interval=8, sink_tokens=2, recent=4)
    k = torch.randn(1, 2, 40, D, device="cuda").to(BF)
    ad.build_cache(k[:, :, :39], k[:, :, :39])
    ad.append(k[:, :, 39], k[:, :, 39])  # full: the next append evicts first
    before = [x.clone() for x in (ad.keys, ad.values, ad.positions, ad.weights, ad.lens, ad.query_pos)]
    for bad in (k[:, :, 0].float(), k[:, :, 0].cpu()):
        with pytest.raises(ValueError, match="tensors on"):
            ad.append(bad, bad)
        assert (ad.length, ad.position, ad.evictions) == (40, 40, 0)
        assert all(torch.equal(a, b) for a, b in zip(before, (ad.keys, ad.values, ad.positions, ad.weights, ad.lens, ad.query_pos)))
    ad.append(k[:, :, 0], k[:, :, 0])
    assert (ad.length, ad.position, ad.evictions) == (33, 41, 1)
    ad.build_cache(k[:, :, :10], k[:, :, :10])
    assert (ad.length, ad.position, ad.evictions) == (10, 10, 0)
    with pytest.raises(ValueError, match="GQA"):
        EvictingCacheAdapter(num_query_heads=0, num_kv_heads=2, budget=32, recent=4)


def test_hook_keeps_nothing_of_a_layer_that_is_gone(monkeypatch):
    from pqhsa_release_b200.pq_hsa_vllm import runtime

    for k, v in {"PQ_HSA_BATCH": "1", "PQ_HSA_ENABLE": "1", "PQ_HSA_DENSE": "1", "PQ_HSA_MULTI_QUERY": "0"}.items():
        monkeypatch.setenv(k, v)
    runtime.reset()
    H, G = 2, 4
    cache = Cache([70, 5, 131], H, BF, 16, "heads")
    q = torch.randn(3, H * G, D, device="cuda").to(BF)
    md = metadata(cache, 1)
    for left in (-1, 3, 20, 50, -1, 9):
        impl = NS(scale=0.1, num_heads=H * G, num_kv_heads=H, sliding_window=(left, 0 if left >= 0 else -1), logits_soft_cap=0, alibi_slopes=None)
        layer, out = object(), torch.zeros_like(q)  # often at the address of the one before
        kv = torch.zeros(3, H, D, dtype=BF, device="cuda")
        runtime.pq_or_dense_forward(None, impl, layer, q, kv, kv, cache.kv, md, output=out)
        o, _, _, tol, _ = ref.attend(cache, q.view(3, 1, H * G, D), scale=0.1, window=left + 1)
        assert ((out.view(3, 1, H * G, D).double() - o).abs() <= tol).all(), left
        del impl, layer
    runtime.reset()


@pytest.mark.parametrize("layout", ["rows", "heads"])
def test_hook_with_a_padded_batch(layout, monkeypatch):
    """Two idle requests (length 0, slot -1) and two rows behind the batch, as a captured step of a fixed size has them."""
    from pqhsa_release_b200.pq_hsa_vllm import runtime

    for k, v in {"PQ_HSA_BATCH": "1", "PQ_HSA_ENABLE": "1", "PQ_HSA_DENSE": "1", "PQ_HSA_MULTI_QUERY": "0"}.items():
        monkeypatch.setenv(k, v)
    runtime.reset()
    H, G = 2, 4
    cache = Cache([70, 0, 131, 0], H, BF, 16, layout)
    g = torch.Generator().manual_seed(3)
    q = torch.randn(6, H * G, D, generator=g).to(BF).cuda()
    k, v = torch.randn(2, 6, H, D, generator=g).to(BF).cuda()
    want = cache.kv.clone()
    for r, n in ((0, 70), (2, 131)):
        for h in range(H):
            cache.put(r, h, n - 1, k[r, h], v[r, h])
    want, cache.kv[:] = cache.kv.clone(), want
    if layout == "heads":  # written before the forward
        cache.kv[:] = want
    slots = [int(cache.table[r, (n - 1) // 16]) * 16 + (n - 1) % 16 if n else -1 for r, n in enumerate(cache.lens)] + [-1, -1]
    md = NS(use_cascade=False, max_query_len=1, num_actual_tokens=4, seq_lens=cache.seq_lens, seq_lens_cpu=cache.seq_lens.cpu(),
            max_seq_len=131, block_table=cache.table, slot_mapping=torch.tensor(slots, device="cuda"))
    impl = NS(scale=0.1, num_heads=H * G, num_kv_heads=H, sliding_window=(-1, -1), logits_soft_cap=0, alibi_slopes=None)
    out = torch.full_like(q, 7.0)
    runtime.pq_or_dense_forward(None, impl, object(), q, k, v, cache.kv, md, output=out)
    assert torch.equal(cache.kv, want)
    o, _, _, tol, _ = ref.attend(cache, q[:4].view(4, 1, H * G, D), scale=0.1)
    assert ((out[:4].view(4, 1, H * G, D).double() - o).abs() <= tol).all()
    assert bool((out[4:] == 7.0).all()) and not bool(out[[1, 3]].any())
    runtime.reset()
