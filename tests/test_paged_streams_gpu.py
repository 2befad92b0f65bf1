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
