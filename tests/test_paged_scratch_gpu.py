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
