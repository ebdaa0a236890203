"""Calls that the documentation of prompts, cache pages and attention over them allows, beside those of every day."""
import pytest
import torch

from helpers import L, pkg
from test_gpu_pages import Model, branches, check_attention, cumulated, extend, filled, ints, new_cache, reference

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def near(out, ref, mass):
    # bf16 rounds to within 2^-8: each probability (the sum divided by is of the unrounded ones) and the output; 1.02
    # covers the fp32 scores and sums
    return ((out.double() - ref).abs() <= 1.02 * 2.0 ** -8 * (mass + ref.abs())).all()


@pytest.mark.parametrize("pitch", [64, 0, 1, 1 << 25])
def test_the_stride_of_a_single_row_is_anything(pitch):
    """torch gives a dim of one any stride: a transposed view's is that of another dim."""
    hq, hk, d = 4, 2, 64
    x = torch.randn(8, d, device="cuda").to(BF)
    q, k, v = (x[a:b].as_strided((1, b - a, d), (pitch, d, 1), x[a:b].storage_offset()) for a, b in ((0, 4), (4, 6), (6, 8)))
    flat = torch.zeros(hq, d, dtype=BF, device="cuda")
    out = flat.as_strided((1, hq, d), (pitch, d, 1))
    pkg.kernels.make_prompt_attention_kernel(hq, hk, d, 0.125)(q, k, v, ints([0, 1]), out)
    assert torch.equal(flat, x[6:8].repeat_interleave(2, 0))
    c = pkg.PageCache(1, 4, 16, hk, d, 2, 2)
    c.reserve(ints([1]), ints([0, 1]))
    c.write(0, k, v, ints([1]), ints([0, 1]))
    flat.zero_()
    pkg.make_prefix_attention_kernel(c, hq, 0.125, 1, 0, 16)(0, q, ints([1]), None, None, out)
    c.check()
    assert torch.equal(flat, x[6:8].repeat_interleave(2, 0))
    turned = x[:4].unsqueeze(1).transpose(0, 1)    # [1, 4, 64], as a projection's heads come
    assert turned.stride(0) == 64
    pkg.make_prefix_attention_kernel(c, hq, 0.125, 1, 0, 16)(0, turned, ints([1]), None, None, out)
    assert torch.equal(flat, x[6:8].repeat_interleave(2, 0))


@pytest.mark.parametrize("bounds,rows", [([0, 3, 8], 7), ([0, 3, 8], 1), ([-2, 3, 8], 8)])
def test_a_write_of_fewer_rows_than_its_tokens_is_reported(bounds, rows):
    """Those that are there are written, the others' slots stay as they were, and check() says so."""
    c = new_cache()
    m = Model(c)
    counts = [bounds[1] - bounds[0], 5]
    c.reserve(ints([2, 0]), cumulated(counts))
    m.reserve([2, 0], counts)
    c.check()
    k = torch.randn(rows, 2, 64, device="cuda").to(BF)
    c.write(1, k, -k, ints([2, 0]), ints(bounds))
    assert int(c.status) == L.PAGES_BAD_ENTRY
    for s, at in ((2, bounds[0]), (0, 3)):
        for pos in range(m.lens[s]):
            if 0 <= at + pos < rows:
                p, slot = m.tables[s][pos // 16], pos % 16
                m.k[1, p, :, slot], m.v[1, p, :, slot] = k[at + pos].cpu(), -k[at + pos].cpu()
    m.check(c)
    with pytest.raises(L.OasisError, match="row"):
        c.check()
    spare = torch.randn(20, 2, 64, device="cuda").to(BF)     # more rows than tokens are none of its business
    c.write(1, spare, -spare, ints([2, 0]), cumulated(counts))
    c.check()


@pytest.mark.parametrize("bad", [-1, 40, 1 << 30])
@pytest.mark.parametrize("copy", [False, True])
def test_a_fork_passes_on_a_page_that_is_not_there(copy, bad):
    """The child is what the parent is, that entry included, no page is lost on it, and check() names the call."""
    c = new_cache()
    m = Model(c)
    extend(c, [0, 1], [70, 20], model=m)
    was = m.tables[0][2]
    c.tables[0, 2] = bad
    c.fork(ints([0, 1]), ints([5, 3]), copy=copy)
    m.fork([0, 1], [5, 3], copy)
    m.refs[m.tables[5][2]] -= 1           # nobody is on the page that the entry would have named
    m.tables[0][2] = m.tables[5][2] = bad
    if copy:                              # nor is it copied to
        lost = [p for p in range(40) if p not in m.tables[0] + m.tables[1] + m.tables[5] + m.tables[3] + [was]]
        for pool, was_pool in ((m.k, c.k), (m.v, c.v)):
            pool[:, lost] = was_pool[:, lost].cpu()
    m.check(c)
    with pytest.raises(L.OasisError, match="fork"):
        c.check()
    c.truncate(ints([5]))
    assert int(c.status) == L.PAGES_BAD_ENTRY and int(c.lens[5]) == 0
    with pytest.raises(L.OasisError):
        c.check()
    c.tables[0, 2] = was
    m.tables[0][2] = was
    m.tables[5][2] = was
    m.refs[was] += 1
    m.truncate([5], [0])
    m.check(c)
    assert extend(c, [5, 6, 7, 8, 9, 10, 11], [80] * 6 + [16 * (len(m.free()) - 30)], model=m) == 0     # all free pages can be had
    m.check(c)


def test_calls_of_more_sequences_than_a_workgroup_plans_at_a_time():
    """Writes that search bounds in memory (1024 sequences on), forks of more than one pass (1024), copies of part-filled pages by
    lists in memory (2048 on): each against the model, in full."""
    import random
    r = random.Random(8)
    c = pkg.PageCache(1, 9001, 16, 1, 64, 2500, 4)
    c.k.zero_()
    c.v.zero_()
    m = Model(c)
    parents = r.sample(range(1300), 1300)
    assert extend(c, parents, [r.choice([0, 1, 5, 16, 33]) for _ in parents], seed=1, model=m) == 0
    m.check(c)
    kids = r.sample(range(1300, 2500), 1200)
    of = [r.randrange(1300) for _ in kids]
    c.fork(ints(of), ints(kids))
    assert m.fork(of, kids, False) == 0
    m.check(c)
    grow = r.sample(range(2500), 2300)
    assert extend(c, grow, [r.choice([0, 1, 1, 2]) for _ in grow], seed=2, model=m) == 0
    m.check(c)
    c.truncate(ints(kids))
    m.truncate(kids, [0] * len(kids))
    c.fork(ints(of), ints(kids), copy=True)
    assert m.fork(of, kids, True) == 0
    m.check(c)
    c.compact()
    m.compact()
    m.check(c)
    c.check()


def test_attention_over_pages_past_32_bits():
    """A layer of 5 GB: own tokens and prefixes of few and of many columns on its last pages, in the second layer."""
    c = pkg.PageCache(2, 40000, 64, 8, 128, 6, 19600)
    c.reserve(ints([0, 1]), ints([0, 39000 * 32, 39000 * 64]))
    extend(c, [2], [300])
    c.fork(ints([2, 2]), ints([3, 4]))
    extend(c, [2, 3, 4, 5], [5, 70, 1, 90], seed=1)
    c.check()
    assert int(c.tables[2:, 0].min()) >= 39000
    check_attention(c, 8, [2, 3, 4, 5], layer=1, max_len=400)
    for heads in (8, 192):
        check_attention(c, heads, [2, 3, 4, 5], [0, 3, 4], [256, 60], layer=1, max_len=400)
    check_attention(c, 8, [5, 2], layer=0, max_len=400)


def overlaps(span, like):
    """Whether the allocator gives out any of the memory [first, last) for tensors of a size."""
    got = [torch.empty_like(like) for _ in range(8)]
    return any(t.data_ptr() < span[1] and span[0] < t.data_ptr() + t.numel() * t.element_size() for t in got)


def busy(stream):
    with torch.cuda.stream(stream):
        torch.cuda._sleep(200_000_000)    # some tenths of a second


def test_memory_of_a_kernel_or_cache_dropped_while_another_stream_uses_it_is_not_given_out():
    """As for any tensor that its stream has been told of: the workspace is nobody's to tell of but the kernel's."""
    c, cu = branches([300], [[3, 50, 7, 0]], 16, 2, 64)
    side = torch.cuda.Stream()
    q = torch.randn(4, 4, 64, device="cuda").to(BF)
    out = torch.zeros_like(q)
    args = ints(range(4)), ints(cu), ints([300])
    torch.cuda.synchronize()
    f = pkg.make_prefix_attention_kernel(c, 4, 0.125, 4, 1, 400)
    workspace = next(x.cell_contents for x in f.__closure__ if torch.is_tensor(x.cell_contents))
    like, span = torch.empty_like(workspace, device="meta"), (workspace.data_ptr(), workspace.data_ptr() + workspace.numel())
    like = torch.empty(like.shape, dtype=like.dtype, device="cuda")
    busy(side)
    with torch.cuda.stream(side):
        f(0, q, *args, out)
    del f, workspace
    assert not side.query() and not overlaps(span, like)
    side.synchronize()
    assert near(out, *reference(c, 0, q, range(4), 0.125))

    d = pkg.PageCache(1, 30, 16, 2, 64, 4, 8)
    spans = [(t, (t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())) for t in (d.k, d.refs, d._work)]
    spans = [(torch.empty_like(t), s) for t, s in spans]
    torch.cuda.synchronize()
    busy(side)
    one, step = ints([1]), ints([0, 9])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        d.reserve(one, step)
    del d
    assert not side.query() and not any(overlaps(s, t) for t, s in spans)
    side.synchronize()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_a_query_that_is_not_finite_reaches_no_other_row_or_head(what, d):
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(300, h, d, generator=g).to(BF).cuda() for h in (4, 2, 2))
    f, cu = pkg.kernels.make_prompt_attention_kernel(4, 2, d, 0.1), ints([0, 170, 300])
    clean, out = torch.zeros_like(q), torch.zeros_like(q)
    f(q, k, v, cu, clean)
    q[100, 1, 3] = q[299, 2, 7] = what
    f(q, k, v, cu, out)
    for row, head in ((100, 1), (299, 2)):
        assert out[row, head].isnan().all()
        out[row, head] = clean[row, head]
    # each within the bound of `near`, whose mass is at most the largest value
    assert ((out.double() - clean.double()).abs() <= 2 * 1.02 * 2.0 ** -8 * (v.abs().max().item() + clean.double().abs())).all()
    for heads, own in ((4, [[20, 0, 70], [5, 6]]), (96, [[20, 0, 70, 9], [5, 6]])):     # few and many columns
        c, cu = branches([208, 100], own, 16, 2, d)
        n = cu[-1]
        a = pkg.make_prefix_attention_kernel(c, heads, 0.1, n, 2, 300)
        q = torch.randn(n, heads, d, generator=g).to(BF).cuda()
        out = torch.zeros_like(q)
        ref, mass = reference(c, 0, q, range(n), 0.1)
        q[1, 1, 3] = q[4, 2, 7] = what
        a(0, q, ints(range(n)), ints(cu), ints([208, 100]), out)
        for row, head in ((1, 1), (4, 2)):
            assert out[row, head].isnan().all()
            out[row, head], ref[row, head] = 0, 0
        # not the same bits: the maximum of a wave's other queries moves when one of them has none
        assert near(out, ref, mass)


def test_rows_of_one_sequence_in_one_group_and_out_of_order():
    """The same sequence in several rows, groups whose rows' sequences are in any order, and rows before and behind all groups."""
    c, cu = branches([96, 48], [[20, 7, 0, 33], [5, 60]], 16, 2, 64)
    check_attention(c, 8, [5, 3, 0, 3, 2, 1, 4, 5, 4, 0], [1, 6, 9], [96, 48])
