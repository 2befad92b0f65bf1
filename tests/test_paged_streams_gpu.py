"""Layers made on one stream, or during a capture, and used on another."""

import pytest
import torch

import paged_ref as ref
from paged_ref import D, Cache
from test_paged_attention_gpu import check, layer, queries

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("given", [F32, torch.float64], ids=["as_kept", "converted"])
def test_slopes_of_a_layer_made_on_a_busy_stream(given):
    cache = Cache([300, 40], 2, BF, 16, "heads")
    q = queries(cache, 4, 1)
    slopes = torch.exp2(-torch.arange(1, 9, device="cuda").to(given))
    want = ref.attend(cache, q, slopes=slopes)
    busy, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(busy):
        for _ in range(4):  # what the allocator hands out next on that stream holds these
            junk = [torch.full((8,), 50.0, device="cuda") for _ in range(4)]
            del junk
    torch.cuda.synchronize()
    with torch.cuda.stream(busy):
        torch.cuda._sleep(50_000_000)
        att = layer(cache, 4, alibi_slopes=slopes)
    with torch.cuda.stream(other):
        out = att.forward(q, cache.seq_lens)
    torch.cuda.synchronize()
    check(out, None, want)


def test_slopes_of_a_layer_made_during_a_capture():
    cache = Cache([300, 40], 2, BF, 16, "heads")
    q = queries(cache, 4, 1)
    slopes = torch.exp2(-torch.arange(1, 9, device="cuda").float())
    want = ref.attend(cache, q, slopes=slopes)
    g, one = torch.cuda.CUDAGraph(), torch.zeros(1, device="cuda")
    with torch.cuda.graph(g):
        one.add_(1.0)
        att = layer(cache, 4, alibi_slopes=slopes)
        captured = att.forward(q, cache.seq_lens)
        with pytest.raises(RuntimeError, match="capture"):
            layer(cache, 4, alibi_slopes=slopes.double())
    check(att.forward(q, cache.seq_lens), None, want)  # before the graph has ever run
    g.replay()
    torch.cuda.synchronize()
    check(captured, None, want)
    check(att.forward(q, cache.seq_lens), None, want)


def test_a_layers_slopes_are_a_copy():
    cache = Cache([300, 40], 2, BF, 16, "heads")
    q = queries(cache, 4, 1)
    slopes = torch.exp2(-torch.arange(1, 9, device="cuda").float())
    want = ref.attend(cache, q, slopes=slopes)
    att = layer(cache, 4, alibi_slopes=slopes)
    slopes.fill_(3.0)
    check(att.forward(q, cache.seq_lens), None, want)


@pytest.mark.parametrize("layout", ["rows", "heads"])
@pytest.mark.parametrize("T", [1, 3])
def test_the_hooks_dense_steps_of_two_layers_in_one_graph(layout, T, monkeypatch):
    """Captured on their first call; replays follow lengths, block tables, rows and queries, and an eager step between
    replays leaves them alone."""
    from types import SimpleNamespace as NS

    from pqhsa_release_b200.pq_hsa_vllm import runtime

    for k, v in {"PQ_HSA_BATCH": "1", "PQ_HSA_ENABLE": "1", "PQ_HSA_DENSE": "1", "PQ_HSA_MULTI_QUERY": "0"}.items():
        monkeypatch.setenv(k, v)
    runtime.reset()
    H, G, n = 2, 4, 3
    caches = [Cache([70, 9, 131], H, BF, 16, layout, seed=s, room=160) for s in (1, 2)]
    lens, table = caches[0].seq_lens, caches[0].table
    for c in caches[1:]:
        c.seq_lens, c.table = lens, table
    impls = [NS(scale=0.1 * (i + 1), num_heads=H * G, num_kv_heads=H, sliding_window=w, logits_soft_cap=cap, alibi_slopes=None)
             for i, (w, cap) in enumerate((((39, 0), 15.0), ((-1, -1), 0)))]
    md = NS(use_cascade=False, max_query_len=T, num_actual_tokens=n * T, seq_lens=lens, max_seq_len=160, block_table=table)
    q = [torch.zeros(n * T, H * G, D, dtype=BF, device="cuda") for _ in caches]
    k, v = ([torch.zeros(n * T, H, D, dtype=BF, device="cuda") for _ in caches] for _ in range(2))
    out = [torch.zeros_like(x) for x in q]

    def step():
        for i, c in enumerate(caches):
            runtime.pq_or_dense_forward(None, impls[i], object(), q[i], k[i], v[i], c.kv, md, output=out[i])

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    g = torch.Generator(device="cuda").manual_seed(3)
    for now in ([70, 9, 131], [71, 12, 0], [5, 160, 33], [3, 3, 3]):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        table.copy_(torch.randperm(caches[0].kv.shape[1 if layout == "rows" else 0], generator=g, device="cuda")[: table.numel()].view_as(table))
        for i, c in enumerate(caches):
            c.lens = now
            for x in (q[i], k[i], v[i]):
                x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
            for r, m in enumerate(now):
                for t in range(T if m else 0):
                    for h in range(H):
                        c.put(r, h, m - T + t, k[i][r * T + t, h], v[i][r * T + t, h])
        want = [ref.attend(c, x.view(n, T, H * G, D), scale=0.1 * (i + 1), softcap=15.0 if i == 0 else 0.0, window=40 if i == 0 else 0)
                for i, (c, x) in enumerate(zip(caches, q))]
        filled = [c.kv.clone() for c in caches]
        if layout == "rows":  # the older pages get the step's rows from the hook
            for c in caches:
                for r, m in enumerate(now):
                    for t in range(T if m else 0):
                        c.put(r, slice(None), m - T + t, torch.zeros(D, dtype=BF), torch.zeros(D, dtype=BF))
        for eager in (False, True, False):
            for o in out:
                o.fill_(9.0)
            step() if eager else graph.replay()
            torch.cuda.synchronize()
            for c, o, w, f in zip(caches, out, want, filled):
                assert torch.equal(c.kv, f)
                check(o.view(n, T, H * G, D), None, w)
    runtime.reset()
