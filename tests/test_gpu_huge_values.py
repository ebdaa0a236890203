"""Values near the ends of bf16's range: what they come to is in range, so no sum on the way may leave it. Against fp64."""
import random

import pytest
import torch

from helpers import pkg
from test_gpu_pages import branches, filled, ints, reference

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
SIZES = [2.0 ** 126, 2.0 ** 110, 2.0 ** -80]    # of the largest value; 2^126 times 1.99 is the last binade but one


def draw(shape, size, seed):
    """Values up to `size` and on one side of zero, so that sums grow with their number."""
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(shape, generator=g, dtype=torch.float64) * 0.9 + 0.1).mul(size * 1.99).to(BF).cuda()


def check(out, ref, mass):
    # as in the tests of ordinary values: bf16 rounds each probability and the output to within 2^-8; 1.02 covers the fp32
    # scores and sums
    assert torch.isfinite(out).all()
    assert ((out.double() - ref).abs() <= 1.02 * 2.0 ** -8 * (mass + ref.abs())).all()


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("spread", [0.0, 1.5])    # of the scores
@pytest.mark.parametrize("heads,kv,d,lens", [(2, 1, 64, [3000]), (2, 2, 128, [1, 700, 64, 129])])
def test_prompts(heads, kv, d, lens, spread, size):
    g = torch.Generator().manual_seed(1)
    n = sum(lens)
    q, k = (torch.randn(n, h, d, generator=g).mul_(spread).to(BF).cuda() for h in (heads, kv))
    v, out = draw((n, kv, d), size, 2), torch.zeros_like(q)
    cu = ints([sum(lens[:i]) for i in range(len(lens) + 1)])
    pkg.kernels.make_prompt_attention_kernel(heads, kv, d, d ** -0.5)(q, k, v, cu, out)
    at = 0
    for x in lens:
        hidden = torch.ones(x, x, dtype=torch.bool, device="cuda").triu(1)
        for h in range(heads):
            s = q[at:at + x, h].double() @ k[at:at + x, h * kv // heads].double().t().contiguous() * d ** -0.5
            ref = s.masked_fill(hidden, -float("inf")).softmax(-1) @ v[at:at + x, h * kv // heads].double()
            check(out[at:at + x, h], ref, ref)
        at += x


def attend(c, heads, rows, cu, prefix, size, spread=1.5):
    g = torch.Generator(device="cuda").manual_seed(5)
    c.k.normal_(generator=g)
    c.k.mul_(spread)
    c.v.copy_(draw(c.v.shape, size, 3))
    q = torch.randn(rows, heads, c.head_dim, generator=g, device="cuda").to(BF)
    out = torch.zeros_like(q)
    f = pkg.make_prefix_attention_kernel(c, heads, c.head_dim ** -0.5, rows, len(prefix) if prefix else 0, int(c.lens.max()))
    f(0, q, ints(list(range(rows))), cu and ints(cu), prefix and ints(prefix), out)
    return out, *reference(c, 0, q, range(rows), c.head_dim ** -0.5)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("spread", [0.0, 1.5])
@pytest.mark.parametrize("rows,hk,heads,d,own", [(2, 1, 2, 64, 4000), (3, 1, 1, 128, 900), (64, 16, 16, 64, 500), (300, 4, 4, 64, 60)])
def test_own_tokens(rows, hk, heads, d, own, spread, size):
    r = random.Random(rows)
    c = filled([r.randint(own // 2, own) for _ in range(rows)], 16, hk, d)
    check(*attend(c, heads, rows, None, None, size, spread))


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("spread", [0.0, 1.5])
@pytest.mark.parametrize("rows,hk,heads,d", [(4, 1, 2, 64), (40, 1, 4, 128), (600, 16, 16, 64)])
def test_prefixes_and_own_tokens(rows, hk, heads, d, spread, size):
    r = random.Random(rows)
    prefix = [r.randint(500, 900), r.randint(100, 300)]
    c, cu = branches(prefix, [[r.randint(0, 40) for _ in range(rows // 2)] for _ in prefix], 16, hk, d)
    # what rows share is read through the first one's pages: the part-filled one behind whole pages is each row's own copy
    prefix = [p // 16 * 16 for p in prefix]
    check(*attend(c, heads, rows, cu, prefix, size, spread))
    assert c.lens.tolist()[0] > prefix[0]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("heads", [2, 40])
def test_rows_that_are_summed_key_by_key(heads, size):
    c, cu = branches([608], [[30, 20, 4]], 16, 1, 64)
    c.truncate(ints([1]), ints([470]))
    seen = draw(c.v.shape, size, 3)
    out, ref, mass = attend(c, heads, 3, cu, [608], size)
    check(out, ref, mass)
    c.v[0, int(c.tables[0, 500 // 16]), 0, 500 % 16] = float("nan")
    again = torch.zeros_like(out)
    g = torch.Generator(device="cuda").manual_seed(5)
    torch.empty_like(c.k).normal_(generator=g)
    q = torch.randn(3, heads, 64, generator=g, device="cuda").to(BF)
    pkg.make_prefix_attention_kernel(c, heads, 0.125, 3, 1, 700)(0, q, ints([0, 1, 2]), ints(cu), ints([608]), again)
    assert again[[0, 2]].isnan().all()
    check(again[1], ref[1], mass[1])
    assert seen.isfinite().all()
