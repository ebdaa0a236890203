"""A K/V cache of pages that sequences share, and attention of single tokens against it.

``PageCache`` holds the pages and their bookkeeping in device memory, so a step of a serving loop (reserve, write each
layer, attend, cut) runs without the host waiting and can be captured into a graph. A refused call (no free pages, a
sequence that is not there) sets bits in ``status`` and changes nothing; the calls after it do nothing either, until
``check`` has raised for it.

No counterpart in the reference, whose cache is the one past frame of a stream (oasis_inference.py:1354-1403).
"""
import ctypes

import torch

from . import _lib as L
from .kernels import Streams, check_heads, check_ints, launch

REFUSALS = {L.PAGES_FULL: "too few free pages",
            L.PAGES_BAD_CALL: "a reserve or fork named a sequence that is not there, twice, or not empty, or too many tokens",
            L.PAGES_BAD_ENTRY: "a truncate or write skipped a sequence, length, page or row that is not there, "
                               "or a fork passed a page on that is not there"}


class PageCache:
    """n_pages pages of page_size tokens (a multiple of 16) for up to max_seqs sequences of up to max_pages pages.

    k, v [n_layers, n_pages, n_kv_heads, page_size, head_dim] (bf16); refs [n_pages], tables [max_seqs, max_pages]
    (page numbers, then -1), lens [max_seqs] and status [1] (int32), all on the device. head_dim is 64 or 128.

    The methods take int32 device vectors (``seqs``: sequence numbers, ``cu``: [sequences + 1], the new tokens of
    seqs[i] being cu[i + 1] - cu[i]) and enqueue on the current stream; calls on one cache must be in order (one
    stream, or events between them)."""

    def __init__(self, n_layers, n_pages, page_size, n_kv_heads, head_dim, max_seqs, max_pages, device="cuda"):
        dev = torch.device(device)
        sizes = n_layers, n_pages, page_size, n_kv_heads, head_dim, max_seqs, max_pages
        # a call of no sequences looks at the sizes and at no memory
        L.call("oasis_pages_truncate", ctypes.byref(L.PageCache(*[16] * 7, *sizes)), None, None, 0, None)
        work = L.count("oasis_pages_work", n_pages, max_seqs)
        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        self.n_layers, self.page_size, self.n_kv_heads, self.head_dim = n_layers, page_size, n_kv_heads, head_dim
        self.k = torch.empty(shape, dtype=torch.bfloat16, device=dev)  # slots of no token may hold anything
        self.v = torch.empty(shape, dtype=torch.bfloat16, device=dev)
        self.device = dev = self.k.device
        self.refs = torch.zeros(n_pages, dtype=torch.int32, device=dev)
        self.tables = torch.full((max_seqs, max_pages), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(max_seqs, dtype=torch.int32, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self._work = torch.empty(work, dtype=torch.int32, device=dev)
        p = [t.data_ptr() for t in (self.k, self.v, self.refs, self.tables, self.lens, self.status, self._work)]
        self.struct = L.PageCache(*p, *sizes)
        self._ref = ctypes.byref(self.struct)
        self._dev = self.refs.get_device()
        self._streams = Streams(self._dev, self.k, self.v, self.refs, self.tables, self.lens, self.status, self._work)

    def _launch(self, name, *args):
        self._streams.used(launch(self._dev, name, self._ref, *args))

    def _lists(self, what, seqs, cu):
        check_ints(what, self._dev, seqs, cu)
        if cu.numel() != seqs.numel() + 1:
            raise L.OasisError(what, -2, "%d sequences and %d bounds" % (seqs.numel(), cu.numel()))

    def reserve(self, seqs, cu):
        """Room for the new tokens of seqs (distinct): lengths grow, the lowest free pages join the tables, a part-filled
        last page that others share is replaced by a copy, for each of them that is named."""
        self._lists("reserve", seqs, cu)
        self._launch("oasis_pages_reserve", seqs.data_ptr(), cu.data_ptr(), seqs.numel())

    def write(self, layer, k, v, seqs, cu):
        """The keys and values [rows, n_kv_heads, head_dim] of the tokens reserved last with the same seqs and cu."""
        self._lists("write", seqs, cu)
        rows = k.shape[0]
        ld_k = check_heads("write", k, rows, self.n_kv_heads, self.head_dim, self._dev)
        ld_v = check_heads("write", v, rows, self.n_kv_heads, self.head_dim, self._dev)
        self._launch("oasis_pages_write", layer, k.data_ptr(), ld_k, v.data_ptr(), ld_v, seqs.data_ptr(), cu.data_ptr(),
                     seqs.numel(), rows)

    def fork(self, parents, children, copy=False):
        """Each empty sequence children[i] (distinct) becomes what parents[i] is, on the same pages, or with copy on free
        pages of its own."""
        check_ints("fork", self._dev, parents, children)
        if parents.numel() != children.numel():
            raise L.OasisError("fork", -2, "%d parents and %d children" % (parents.numel(), children.numel()))
        self._launch("oasis_pages_fork", parents.data_ptr(), children.data_ptr(), parents.numel(), bool(copy))

    def truncate(self, seqs, keep=None):
        """Cuts seqs to their first keep[i] tokens (none by default); pages that no sequence is left on become free."""
        check_ints("truncate", self._dev, seqs, *(() if keep is None else (keep,)))
        if keep is not None and keep.numel() != seqs.numel():
            raise L.OasisError("truncate", -2, "%d sequences and %d lengths" % (seqs.numel(), keep.numel()))
        self._launch("oasis_pages_truncate", seqs.data_ptr(), None if keep is None else keep.data_ptr(), seqs.numel())

    def compact(self):
        """Moves the pages in use to the lowest numbers; tables and references follow."""
        self._launch("oasis_pages_compact")

    def check(self):
        """Waits for the calls so far; raises OasisError if one was refused, and clears the refusal."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise L.OasisError("PageCache", -5, "; ".join(m for b, m in REFUSALS.items() if bits & b))


def make_prefix_attention_kernel(cache, n_heads, scale_val, max_rows, max_groups, max_len):
    """Attention of one query token of each of up to max_rows sequences against their pages in ``cache``, the tokens
    that the sequences of a group share read once for all of them.

    The kernel takes layer, q [rows, n_heads, head_dim] (bf16), seqs [rows], cu_groups [groups + 1] and prefix_lens
    [groups] (rows cu_groups[g] .. cu_groups[g + 1] - 1 begin with the same prefix_lens[g] tokens; None for both where
    nothing is shared), and out like q, which overlaps none of them. max_len: about how many tokens the longest sequence has.
    The prefixes are read together where there are fewer groups than rows, whatever the groups' bounds are: groups without
    rows, as in vectors padded to a fixed size, give right results and cost the sharing.

    The workspace is the kernel's own: its calls must not overlap, nor graphs that hold them, which need it as long as they
    are replayed."""
    work = L.count("oasis_pages_attention_workspace", max_rows, max_groups, max_len, n_heads, cache.n_kv_heads,
                   cache.head_dim)
    workspace = torch.empty(work, dtype=torch.uint8, device=cache.device)

    dev, dim, at = cache._dev, cache.head_dim, workspace.data_ptr()
    streams = Streams(dev, workspace)

    def prefix_attention_kernel(layer, q, seqs, cu_groups, prefix_lens, out):
        if (cu_groups is None) != (prefix_lens is None):
            raise L.OasisError("prefix_attention", -1, "cu_groups and prefix_lens come together, or neither")
        rows = q.shape[0]
        ld_q = check_heads("prefix_attention", q, rows, n_heads, dim, dev)
        ld_out = check_heads("prefix_attention", out, rows, n_heads, dim, dev)
        check_ints("prefix_attention", dev, seqs)
        groups = 0
        if cu_groups is not None:
            check_ints("prefix_attention", dev, cu_groups, prefix_lens)
            groups = prefix_lens.numel()
            if cu_groups.numel() != groups + 1:
                raise L.OasisError("prefix_attention", -2, "%d groups and %d bounds" % (groups, cu_groups.numel()))
        if seqs.numel() != rows or rows > max_rows or groups > max_groups:
            raise L.OasisError("prefix_attention", -2, "%d rows of %d sequences in %d groups; the kernel was made for %d and %d"
                               % (rows, seqs.numel(), groups, max_rows, max_groups))
        stream = launch(dev, "oasis_pages_attention", cache._ref, layer, q.data_ptr(), ld_q, out.data_ptr(), ld_out,
                        seqs.data_ptr(), rows, cu_groups.data_ptr() if groups else None,
                        prefix_lens.data_ptr() if groups else None, groups, max_len, n_heads, scale_val, at, workspace.numel())
        streams.used(stream)
        cache._streams.used(stream)
    return prefix_attention_kernel
