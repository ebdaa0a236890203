"""What the Python surface of prompts and cache pages refuses or takes on the host, before any device work."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from helpers import L, pkg

BF = torch.bfloat16
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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


@pytest.mark.parametrize("change,needle", [
    (dict(page_size=24), "page_size"), (dict(page_size=2048), "page_size"), (dict(head_dim=96), "head_dim"), (dict(max_seqs=65537), "shape"),
    (dict(n_layers=0), "shape"), (dict(n_kv_heads=-1), "shape"), (dict(max_pages=0), "shape"), (dict(max_seqs=-3), "shape"), (dict(n_pages=0), "shape")])
def test_a_cache_of_sizes_that_no_call_takes_is_refused_before_its_pools_are_allocated(change, needle):
    sizes = dict(n_layers=60000, n_pages=1 << 27, page_size=16, n_kv_heads=1000, head_dim=64, max_seqs=4, max_pages=8)
    with pytest.raises(L.OasisError, match=needle):
        pkg.PageCache(**(sizes | change), device="cpu")     # pools past all memory


def test_the_package_imports_where_torch_has_no_device_backend():
    """As before the serving calls: their way to the current stream is looked for when the first of them launches."""
    code = """
import torch
for name in [n for n in vars(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
from __graft_entry__ import load_package
pkg = load_package()
assert pkg.PageCache(1, 4, 16, 2, 64, 2, 2, device="cpu").page_size == 16
print("imported")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "imported" in r.stdout, r.stderr[-2000:]


def test_scratch_sizes_that_are_refused_say_so():
    for args in ((0, 7), (7, 0), (-1, 1)):
        assert L.lib().oasis_pages_reserve(None, None, None, 1, None) < 0      # another message is the last
        with pytest.raises(L.OasisError, match="%d pages and %d sequences" % args):
            L.count("oasis_pages_work", *args)


FAKE = ctypes.c_void_p(0x1000)
SHAPE = -2


def cache(**kw):
    a = dict(k=16, v=16, refs=16, tables=16, lens=16, status=16, work=16, n_layers=2, n_pages=10, page_size=16, n_kv_heads=2, head_dim=64,
             max_seqs=65536, max_pages=8) | kw
    return ctypes.byref(L.PageCache(*a.values()))


@pytest.mark.parametrize("name,args,needle", [
    ("oasis_prompt_attention", (FAKE, 64, FAKE, 64, FAKE, 64, FAKE, 64, FAKE, 65537, 1 << 20, 1, 1, 64, 0.1, None), "count"),
    # 2^16 + 2^12 tiles of 128 heads, more than one launch has
    ("oasis_prompt_attention", (FAKE, 8192, FAKE, 8192, FAKE, 8192, FAKE, 8192, FAKE, 65536, 1 << 20, 128, 128, 64, 0.1, None), "tiles"),
    ("oasis_pages_write", (cache(), 0, FAKE, 128, FAKE, 128, FAKE, FAKE, 1, 1 << 26, None), "count"),
    ("oasis_pages_attention", (cache(n_kv_heads=1024), 0, FAKE, 65536, FAKE, 65536, FAKE, 65536, None, None, 0, 5000, 1024, 0.1, FAKE, 1 << 40,
                               None), "parts"),
    ("oasis_pages_attention", (cache(n_kv_heads=1024), 0, FAKE, 65536, FAKE, 65536, FAKE, 65536, FAKE, FAKE, 60000, 5000, 1024, 0.1, FAKE,
                               1 << 50, None), "parts")])
def test_calls_of_more_workgroups_than_a_launch_has_are_refused(name, args, needle):
    """A launch has less than 2^32 threads."""
    h = L.lib()
    rc = getattr(h, name)(*args)
    assert rc == SHAPE and needle in h.oasis_last_error().decode(), (rc, h.oasis_last_error())


def test_a_scale_whose_product_with_log2_e_is_infinite_is_refused():
    h = L.lib()
    for scale, refused in ((3e38, True), (2.36e38, True), (float("inf"), True), (2.3e38, False)):
        for name, args in (("oasis_prompt_attention", (None, 64, FAKE, 64, FAKE, 64, FAKE, 64, FAKE, 1, 1, 1, 1, 64, scale, None)),
                           ("oasis_pages_attention", (cache(), 0, None, 128, FAKE, 128, FAKE, 1, None, None, 0, 10, 2, scale, None, 0, None))):
            rc = getattr(h, name)(*args)
            assert rc == (-5 if refused else -1) and ("scale" if refused else "null") in h.oasis_last_error().decode(), (name, scale)
