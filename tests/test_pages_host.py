"""What the Python surface of prompts and cache pages refuses or takes on the host, before any device work."""
import pytest
import torch

from helpers import L, pkg

BF = torch.bfloat16


def test_no_call_launches_on_a_cache_in_host_memory():
    c = pkg.PageCache(1, 4, 16, 2, 64, 2, 2, device="cpu")
    one, cu = torch.zeros(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    k = torch.zeros(1, 2, 64, dtype=BF)
    for call in (c.compact, lambda: c.truncate(one), lambda: c.reserve(one, cu), lambda: c.fork(one, one), lambda: c.write(0, k, k, one, cu)):
        with pytest.raises(L.OasisError, match="device"):
            call()


def test_group_bounds_and_prefix_lengths_come_together():
    c = pkg.PageCache(1, 4, 16, 2, 64, 2, 2, device="cpu")
    f = pkg.make_prefix_attention_kernel(c, 2, 0.125, 2, 1, 16)
    q, two = torch.zeros(2, 2, 64, dtype=BF), torch.zeros(2, dtype=torch.int32)
    for bounds, prefix in ((two, None), (None, two[:1])):
        with pytest.raises(L.OasisError, match="together"):
            f(0, q, two, bounds, prefix, q)
