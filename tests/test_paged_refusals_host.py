"""More refusals of the dense paged operators and the evicting adapter, without a GPU."""

import pytest
import torch

from pqhsa_release_b200 import EvictingCacheAdapter, PagedAttention


def test_no_cpu_path():
    ad = EvictingCacheAdapter(num_query_heads=4, num_kv_heads=2, budget=8, recent=2, sink_tokens=1)
    x = torch.zeros(1, 2, 3, 128)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ad.build_cache(x, x)
    with pytest.raises(RuntimeError, match="build_cache"):
        ad.decode_step(x[:, :, 0].repeat(1, 2, 1), x[:, :, 0], x[:, :, 0])


@pytest.mark.parametrize("kw", [dict(softcap=1e-50), dict(softcap=1e39), dict(scale=1e39), dict(scale=-1e300)])
def test_numbers_that_32_bits_do_not_hold(kw):
    """A cap that rounds to nothing would be no cap."""
    with pytest.raises(ValueError, match="32 bits"):
        PagedAttention(num_query_heads=8, num_kv_heads=2, max_requests=2, token_capacity=64, dtype=torch.bfloat16, device="cuda", **kw)
