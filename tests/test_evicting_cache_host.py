"""What the evicting adapter refuses without a GPU."""

import pytest
import torch

from pqhsa_release_b200 import EvictingCacheAdapter


def test_no_cpu_path():
    ad = EvictingCacheAdapter(num_query_heads=4, num_kv_heads=2, budget=8, recent=2, sink_tokens=1)
    x = torch.zeros(1, 2, 3, 128)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ad.build_cache(x, x)
    with pytest.raises(RuntimeError, match="build_cache"):
        ad.decode_step(x[:, :, 0].repeat(1, 2, 1), x[:, :, 0], x[:, :, 0])
