"""More calls of the dense paged operators that are refused, and leave everything as it was."""

import pytest
import torch

from paged_ref import D, Cache
from test_paged_attention_gpu import layer, queries

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def test_an_out_whose_rows_share_memory():
    cache = Cache([30, 40], 2, BF, 16, "heads")
    att = layer(cache, 4, 2)
    q = queries(cache, 4, 2)
    want = att.forward(q, cache.seq_lens)
    base = torch.full((2, 2, 8, D), 7.0, dtype=BF, device="cuda")
    for out in (base[:1].expand(2, -1, -1, -1), base[:, :1].expand(-1, 2, -1, -1), base[:, :, :1].expand(-1, -1, 8, -1), base[:, :, :, :1].expand(-1, -1, -1, D)):
        with pytest.raises(ValueError, match="out"):
            att.forward(q, cache.seq_lens, out=out)
    assert bool((base == 7.0).all())
    # one row of a dimension has no stride of its own
    one = att.forward(q[:1, :1], cache.seq_lens[:1], out=base[:1, :1].as_strided((1, 1, 8, D), (0, 0, D, 1)))
    assert one.shape == (1, 1, 8, D)
    assert torch.equal(att.forward(q, cache.seq_lens), want)
