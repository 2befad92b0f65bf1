"""Device memory that the dense paged operators take beside the cache: by the call's size, once per stream of execution."""

import ctypes as C
import threading

import pytest
import torch

import paged_ref as ref
from paged_ref import D, Cache
from pqhsa_release_b200 import EvictingCacheAdapter, PagedAttention, _lib
from test_paged_attention_gpu import check, layer, queries

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
MB = 1 << 20


def grown(call, *args, **kw):
    """Bytes on the device after a call that were not there before it, its result kept."""
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    keep = call(*args, **kw)
    torch.cuda.synchronize()
    return torch.cuda.memory_allocated() - before, keep


def test_workspaces_are_sized_by_the_call():
    H, G, cap, B = 2, 4, 8192, 16
    cache = Cache([5, 9] + [0] * (B - 2), H, BF, 16, "heads", room=cap)
    att = layer(cache, G, 8)
    mass = torch.zeros(B, H, cap, device="cuda")
    q = queries(cache, G, 8)
    full = B * H * 8 * G * cap * 4  # scores of the largest call: 32 MB
    out = torch.empty_like(q[:2, :1])
    n, _ = grown(att.forward, q[:2, :1].contiguous(), cache.seq_lens[:2], out=out, mass=mass)
    assert n < full // 64 + 2 * MB
    want = ref.attend(cache, q)
    got = torch.empty_like(q)
    n, _ = grown(att.forward, q, cache.seq_lens, out=got, mass=mass)
    assert full // 2 < n < full + 8 * MB
    check(got, None, want)
    n, _ = grown(att.forward, q[:2, :1].contiguous(), cache.seq_lens[:2], out=out, mass=mass)  # the larger one serves
    assert n == 0
    # calls of growing sizes in one capture, each with the scratch memory it was recorded with
    outs, g = [torch.empty_like(q[:b, 8 - t :]) for b, t in ((1, 1), (2, 4), (16, 8))], torch.cuda.CUDAGraph()
    qs = [q[:b, 8 - t :].contiguous() for b, t in ((1, 1), (2, 4), (16, 8))]
    masses = [torch.zeros_like(mass) for _ in qs]
    with torch.cuda.graph(g):
        for x, o, m in zip(qs, outs, masses):
            att.forward(x, cache.seq_lens[: x.shape[0]], out=o, mass=m)
    for m in masses:
        m.zero_()
    g.replay()
    torch.cuda.synchronize()
    for (b, t), o, m, x in zip(((1, 1), (2, 4), (16, 8)), outs, masses, qs):
        check(o, None, tuple(w[:b, 8 - t :] if torch.is_tensor(w) else w for w in want))
        one = torch.zeros_like(m)
        att.forward(x, cache.seq_lens[:b], mass=one)
        assert torch.equal(one, m)


@pytest.mark.parametrize("S", [2000, 8192], ids=["short", "past_the_budget"])
def test_an_evicting_cache_keeps_the_scratch_of_one_token(S):
    B, H, G, budget, interval = 8, 2, 4, 4096, 256
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF)
    keys, values, wq = r(B, H, S, D), r(B, H, S, D), r(B, H * G, 16, D)
    ad = EvictingCacheAdapter(num_query_heads=H * G, num_kv_heads=H, budget=budget, interval=interval)
    grown(ad.build_cache, keys, values, wq)
    ad.decode_step(r(B, H * G, D), r(B, H, D), r(B, H, D))
    room = budget + interval
    rows = B * H * room
    cache = 2 * rows * D * 2 + 8 * rows  # keys, values, positions, weights
    one = rows * G * 4                    # the scores of a token
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    del ad
    held = before - torch.cuda.memory_allocated()
    evicting = 4 * B * H * (3 * budget + 8) if S > budget else 0
    assert held < cache + one + evicting + 2 * MB, (held - cache) / one


def test_the_layers_of_a_model_share_their_scratch():
    """Sixteen layers of one step, eager and in captures of two sizes: what they hold beside the first layer's is nothing,
    and each layer's results are its own."""
    H, G, B, L = 2, 4, 6, 16
    caches = [Cache([300, 77, 1, 0, 512, 130], H, BF, 16, "heads", seed=s) for s in range(L)]
    qs = [queries(c, G, 1, s) for s, c in enumerate(caches)]
    want = [ref.attend(c, q) for c, q in zip(caches, qs)]
    outs = [torch.empty_like(q) for q in qs]
    layers = [layer(c, G) for c in caches]

    def steps(some, b=B):
        for att, c, q, o in some:
            att.forward(q[:b], c.seq_lens[:b], out=o[:b])

    every = list(zip(layers, caches, qs, outs))
    first, _ = grown(steps, every[:1])
    assert first > 0 and grown(steps, every[1:])[0] == 0
    for o, w in zip(outs, want):
        check(o, None, w)
    graphs = []
    for b in (B, 2):
        before = torch.cuda.memory_allocated()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            steps(every, b)
        graphs.append((g, b, torch.cuda.memory_allocated() - before))
    for g, b, held in graphs:
        assert 0 < held <= first  # one workspace
        for o in outs:
            o.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            check(o[:b], None, tuple(x[:b] if torch.is_tensor(x) else x for x in w))
    # a layer that is gone takes nothing along that the others use
    del layers[0], every[0]
    steps(every)
    torch.cuda.synchronize()
    for o, w in zip(outs[1:], want[1:]):
        check(o, None, w)


def test_two_threads_on_one_stream():
    """An attention with weights is two kernels; another thread's call on the same stream can come between them."""
    H, G = 2, 4
    caches = [Cache([2000, 300], H, BF, 16, "heads", seed=s) for s in (1, 2)]
    qs = [queries(c, G, 1, s) for s, c in enumerate(caches)]
    layers = [layer(c, G) for c in caches]
    masses = [torch.zeros(2, H, c.cap, device="cuda") for c in caches]
    alone = []
    for att, c, q in zip(layers, caches, qs):
        m = torch.zeros(2, H, c.cap, device="cuda")
        att.forward(q, c.seq_lens, mass=m)
        alone.append(m)
    torch.cuda.synchronize()

    def work(i):
        for _ in range(200):
            layers[i].forward(qs[i], caches[i].seq_lens, mass=masses[i])

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for m, one in zip(masses, alone):
        total = torch.zeros_like(m)
        for _ in range(200):
            total += one
        assert torch.equal(m, total)


def test_threads_that_come_and_go_leave_nothing_behind():
    cache = Cache([300, 77], 2, BF, 16, "heads")
    q, want = queries(cache, 4, 1), ref.attend(cache, queries(cache, 4, 1))
    att, out = layer(cache, 4), torch.empty_like(q)
    att.forward(q, cache.seq_lens, out=out)
    gate = threading.Barrier(12)

    def work():
        gate.wait()  # all alive at once: no thread takes over another's identity
        with turn:
            att.forward(q, cache.seq_lens, out=out)

    turn = threading.Lock()

    def all_of_them():
        threads = [threading.Thread(target=work) for _ in range(12)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()

    assert grown(all_of_them)[0] == 0
    check(out, None, want)
