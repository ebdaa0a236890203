"""Keys whose scores are large and nearly equal, met by different waves, in different parts of a sequence and on both sides
of a group's prefix: the weights of sums that were taken apart have to be as exact as those within one. Against fp64."""
import random

import pytest
import torch

from helpers import pkg
from test_gpu_pages import branches, filled, ints, reference

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
SCALE = 0.125
# raw scores: the scaled one in powers of two is 0.18 of them, so these lie around 2^17, 2^19 and up to both sides of 2^20
RAW = [(727_000, 727_100), (2_907_000, 2_907_100), (5_810_000, 5_814_000), (5_813_800, 5_815_200), (8_000_000, 8_000_100)]


def key_of(raw, d):
    """A key whose product with `query` is `raw` (below 2^24), each step of it exact in bf16 and in fp32."""
    k = torch.zeros(d)
    k[0], k[1], k[2] = raw >> 16, raw >> 8 & 255, raw & 255
    return k.to(BF)


def query(rows, heads, d):
    q = torch.zeros(rows, heads, d, dtype=BF)
    q[..., 0], q[..., 1], q[..., 2] = 65536, 256, 1
    return q.cuda()


def plant(c, raws, r, seqs, lens, most=None):
    """Two keys of each sequence have large scores 1 to 5 apart and values of opposite sign, at places that differ; the others
    have a score and value of 0."""
    c.k.zero_()
    c.v.zero_()
    tables = c.tables.tolist()
    for s in seqs:
        base, n = r.randint(*raws), min(lens[s], most or lens[s])
        for at, raw, v in zip(r.sample(range(n), 2), (base, base + r.randint(1, 5)), r.choice([(1.0, -1.0), (-1.0, 1.0)])):
            p, slot = tables[s][at // c.page_size], at % c.page_size
            c.k[0, p, :, slot], c.v[0, p, :, slot] = key_of(raw, c.head_dim).cuda(), v


def check(out, ref, mass):
    # bf16 rounds to within 2^-8: each probability (the sum divided by is of the unrounded ones) and the output; 1.02
    # covers the fp32 sums. The scores and their differences are exact.
    worst = ((out.double() - ref).abs() / (mass + ref.abs()).clamp(min=1e-30)).max().item()
    assert worst <= 1.02 * 2.0 ** -8, worst


def attend(c, heads, rows, cu, prefix, max_len):
    q = query(rows, heads, c.head_dim)
    out = torch.zeros_like(q)
    f = pkg.make_prefix_attention_kernel(c, heads, SCALE, rows, len(prefix) if prefix else 0, max_len)
    f(0, q, ints(list(range(rows))), cu and ints(cu), prefix and ints(prefix), out)
    return out, *reference(c, 0, q, range(rows), SCALE)


@pytest.mark.parametrize("raws", RAW)
@pytest.mark.parametrize("rows,hk,heads,d,own", [
    (3, 1, 1, 64, 3000), (3, 1, 2, 128, 3000),      # parts of a long sequence, eight waves to each
    (64, 16, 16, 64, 500), (64, 16, 16, 128, 300),  # four waves to a row's key head
    (64, 16, 16, 64, 150), (300, 4, 4, 64, 60)])    # two and one
def test_own_tokens(raws, rows, hk, heads, d, own):
    r = random.Random(rows + raws[0])
    lens = [r.randint(own // 2, own) for _ in range(rows)]
    c = filled(lens, 16, hk, d)
    plant(c, raws, r, range(rows), lens)
    check(*attend(c, heads, rows, None, None, own))


# few columns and many of them, in one launch with the rows' own tokens and in one before it
@pytest.mark.parametrize("raws", RAW)
@pytest.mark.parametrize("rows,hk,heads,d", [(4, 1, 2, 64), (4, 1, 2, 128), (40, 1, 4, 64), (40, 1, 4, 128), (300, 16, 16, 64),
                                             (600, 16, 16, 64), (600, 16, 16, 128)])
def test_prefixes_and_own_tokens(raws, rows, hk, heads, d):
    r = random.Random(rows + raws[0])
    groups = 60 if rows == 600 and d == 128 else 2
    prefix = [16 * r.randint(19, 43) for _ in range(groups)]    # whole pages: what is planted in one is in all rows' prefix
    own = [[r.randint(2, 40) for _ in range(rows // groups)] for _ in prefix]
    c, cu = branches(prefix, own, 16, hk, d)
    lens = c.lens.tolist()
    for most in (None, 300):    # two of the row's own and the prefix's keys, and of the prefix's alone
        plant(c, raws, r, range(rows) if most is None else cu[:-1], lens, most)
        if most is None:
            # one of each group's first keys too, as near to the rows' own
            for s in cu[:-1]:
                p = int(c.tables[s, 0])
                c.k[0, p, :, 3], c.v[0, p, :, 3] = key_of(raws[1], d).cuda(), 1.0
        check(*attend(c, heads, rows, cu, prefix, 800))


@pytest.mark.parametrize("raws", RAW)
@pytest.mark.parametrize("heads", [2, 40])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_that_are_summed_key_by_key(raws, heads, d):
    """A value that is not finite behind a row that ends inside the prefix: what that row sees is summed again."""
    r = random.Random(heads + raws[0])
    c, cu = branches([608], [[30, 20, 4]], 16, 1, d)
    c.truncate(ints([1]), ints([470]))
    plant(c, raws, r, range(3), [450] * 3)
    c.v[0, int(c.tables[0, 500 // 16]), 0, 500 % 16] = float("nan")
    out, ref, mass = attend(c, heads, 3, cu, [608], 700)
    check(out[1], ref[1], mass[1])
    assert out[[0, 2]].isnan().all()


@pytest.mark.parametrize("raws", RAW)
@pytest.mark.parametrize("d", [64, 128])
def test_prompts(raws, d):
    """The running maximum moves from tile to tile, over the border where scores are scaled after the difference too."""
    r = random.Random(d + raws[0])
    n = 700
    k, v = torch.zeros(n, 1, d, dtype=BF), torch.zeros(n, 1, d, dtype=BF)
    base = r.randint(*raws)
    for i, at in enumerate(r.sample(range(n), 12)):
        k[at, 0], v[at] = key_of(base + r.randint(0, 60), d), (-1.0) ** i
    k, v, q = k.cuda(), v.cuda(), query(n, 1, d)
    out = torch.zeros_like(q)
    pkg.kernels.make_prompt_attention_kernel(1, 1, d, SCALE)(q, k, v, ints([0, n]), out)
    s = (q[:, 0].double() @ k[:, 0].double().t().contiguous() * SCALE).masked_fill(
        torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -float("inf"))
    p = s.softmax(-1)
    check(out[:, 0], p @ v[:, 0].double(), p @ v[:, 0].double().abs())


def below(n, raws, d, seed):
    """Keys whose scores all lie far below zero, up to 400 apart, and values of both signs."""
    g = torch.Generator().manual_seed(seed)
    raw = torch.randint(raws[0], raws[1], (1,), generator=g) + torch.randint(0, 401, (n,), generator=g)
    k = torch.zeros(n, d)
    k[:, 0], k[:, 1], k[:, 2] = raw >> 16, raw >> 8 & 255, raw & 255    # as key_of
    return k.to(BF).cuda(), (torch.randint(0, 2, (n,), generator=g) * 2 - 1).to(BF).cuda()


@pytest.mark.parametrize("raws", RAW)
@pytest.mark.parametrize("rows,hk,heads,d,shared", [(3, 1, 1, 64, False), (64, 16, 16, 128, False), (4, 1, 2, 64, True), (40, 1, 4, 128, True),
                                                    (600, 16, 16, 64, True)])
def test_scores_far_below_zero(rows, hk, heads, d, shared, raws):
    r = random.Random(rows)
    if shared:
        prefix = [16 * r.randint(19, 43) for _ in range(2)]
        c, cu = branches(prefix, [[r.randint(2, 40) for _ in range(rows // 2)] for _ in prefix], 16, hk, d)
    else:
        prefix, cu = None, None
        c = filled([r.randint(400, 800) for _ in range(rows)], 16, hk, d)
    k, v = below(c.refs.numel() * 16, raws, d, rows + raws[0])
    c.k[0] = k.view(-1, 1, 16, d)
    c.v[0] = v.view(-1, 1, 16, 1)
    q = -query(rows, heads, d)
    out = torch.zeros_like(q)
    f = pkg.make_prefix_attention_kernel(c, heads, SCALE, rows, len(prefix) if prefix else 0, int(c.lens.max()))
    f(0, q, ints(list(range(rows))), cu and ints(cu), prefix and ints(prefix), out)
    check(out, *reference(c, 0, q, range(rows), SCALE))


@pytest.mark.parametrize("raws", RAW)
@pytest.mark.parametrize("d", [64, 128])
def test_prompts_of_scores_far_below_zero(raws, d):
    n = 700
    k, v = below(n, raws, d, d + raws[0])
    q = -query(n, 1, d)
    v = v.view(n, 1, 1).expand(n, 1, d).contiguous()
    out = torch.zeros_like(q)
    pkg.kernels.make_prompt_attention_kernel(1, 1, d, SCALE)(q, k.view(n, 1, d), v, ints([0, n]), out)
    s = (q[:, 0].double() @ k.double().t().contiguous() * SCALE).masked_fill(
        torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -float("inf"))
    p = s.softmax(-1)
    check(out[:, 0], p @ v[:, 0].double(), p @ v[:, 0].double().abs())


@pytest.mark.parametrize("rows,hk,heads,d,lens,shared", [(300, 4, 4, 64, 60, 0), (3, 1, 1, 128, 700, 0), (64, 16, 16, 64, 500, 0), (4, 1, 2, 64, 320, 304),
                                                         (40, 1, 4, 128, 320, 304)])
@pytest.mark.parametrize("gone", [32, 256])
def test_keys_of_minus_infinity_before_scores_far_below_zero(rows, hk, heads, d, lens, shared, gone):
    """Whole tiles that count for nothing, and behind them a row's first finite scores."""
    gone = min(gone, 32 if lens < 300 else 256)
    if shared:
        c, cu = branches([shared], [[lens - shared] * rows], 16, hk, d)
    else:
        c, cu = filled([lens] * rows, 16, hk, d), None
    g = torch.Generator(device="cuda").manual_seed(1)
    c.v.copy_(torch.randn(c.v.shape, generator=g, device="cuda").to(BF))
    c.k.zero_()
    c.k[..., 0] = (torch.randn(c.k.shape[:-1], generator=g, device="cuda") - 3000).to(BF)
    pages = c.tables[:, :gone // 16].flatten().unique().long()
    c.k[:, pages, :, :, 0] = -float("inf")
    q = torch.zeros(rows, heads, d, dtype=BF, device="cuda")
    q[..., 0] = 1
    out = torch.zeros_like(q)
    f = pkg.make_prefix_attention_kernel(c, heads, SCALE, rows, 1 if shared else 0, lens)
    f(0, q, ints(list(range(rows))), ints([0, rows]) if shared else None, ints([shared]) if shared else None, out)
    n = torch.arange(lens, device="cuda")
    for row in (0, rows - 1):
        ids = c.tables[row].long()[n // 16]
        for h in range(heads):
            s = c.k[0, ids, h * hk // heads, n % 16, 0].double() * SCALE
            p, v = s.softmax(0), c.v[0, ids, h * hk // heads, n % 16].double()
            check(out[row, h], p @ v, p @ v.abs())
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("d", [64, 128])
def test_prompts_whose_last_keys_score_minus_infinity(d):
    n = 400
    g = torch.Generator().manual_seed(2)
    k, v, q = (torch.zeros(n, 1, d) for _ in range(3))
    k[:, 0, 0], q[:, 0, 0] = torch.randn(n, generator=g) - 3000, 1
    k[130:, 0, 0] = -float("inf")
    v.copy_(torch.randn(n, 1, d, generator=g))
    q, k, v = (x.to(BF).cuda() for x in (q, k, v))
    out = torch.zeros_like(q)
    pkg.kernels.make_prompt_attention_kernel(1, 1, d, SCALE)(q, k, v, ints([0, n]), out)
    s = (k[:, 0, 0].double() * SCALE).expand(n, n).masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -float("inf"))
    p = s.softmax(-1)
    check(out[:, 0], p @ v[:, 0].double(), p @ v[:, 0].double().abs())
    assert torch.isfinite(out).all()
