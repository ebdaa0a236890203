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
