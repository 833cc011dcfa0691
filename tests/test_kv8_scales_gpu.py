"""Attention over an 8-bit cache whose blocks have scales far apart, against 64 bits, each head by its own largest output.

Tolerance.  The output is rounded to bfloat16 (2**-9 of itself), a weight to fp16 (2**-12 of itself, and 2**-25 of the largest weight in all
of up to 1100 keys), the score of a key is off by 2**-16 of the scores' spread (below 100 here): 2e-3.  An output is a sum of a few weights
times codes of either sign, seldom smaller than a fifth of the largest of its head: 1e-2 of the head's largest output."""
import math

import pytest
import torch

import kv8_refs as R
from test_kv8_gpu import portions_call, rows_call, tiles_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from mlx_lm_b200 import ops as o
    o.require_cuda()
    return o


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


KINDS = ["portions", "rows", "rows float32"]


def check(ops, kind, cache, spans, q, n_heads, scale, window=0, sinks=None):
    pos, req = R.steps(spans)
    want = R.attention(cache, q.cpu(), pos, req, n_heads, scale, window, sinks).view(-1, n_heads, cache.dim)
    top = want.abs().amax(2, keepdim=True)
    if kind == "portions":
        out, status = portions_call(ops, cache, q, tiles_of(spans), n_heads, scale, window, sinks)
    else:
        out, status = rows_call(ops, cache, q if kind == "rows" else q.float(), pos, req, n_heads, scale, window, sinks)
    assert int(status.item()) == 0
    err = (out.double().cpu().view_as(want) - want).abs() / top.clamp(min=1e-30)
    assert float(err.max()) <= 1e-2, float(err.max())
    assert not bool(out.view_as(want)[(top == 0).expand_as(want).cuda()].any())      # nothing but values of 0: exactly 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n_heads,heads,dim", [(4, 2, 64), (3, 3, 64), (4, 2, 128), (2, 2, 48)])
@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-6, 1e-8, 1e-20])
@pytest.mark.parametrize("zeros", ["first", "middle", "many", "last"])
def test_a_block_of_zeros_among_small_values(ops, kind, n_heads, heads, dim, size, zeros):
    spans = [(900, 124)]
    cache = R.Cache([1024], heads, dim, 16, seed=dim)
    cache.vs *= size
    which = {"first": [0], "middle": [31, 32], "many": list(range(0, 64, 3)), "last": [63]}[zeros]
    for i in which:
        cache.vs[int(cache.table[0, i])] = 0.0
    q = (normal(dim, 124, n_heads * dim) * 1.5).bfloat16().cuda()
    sinks = normal(1, n_heads) if zeros == "middle" else None
    check(ops, kind, cache, spans, q, n_heads, 0.25 * (64 / dim) ** 0.5, sinks=sinks)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [0.05, 0.6])          # 0.6: scores of up to 200, beyond what an exponential holds
@pytest.mark.parametrize("window,sinks", [(0, False), (40, True)])
def test_rows_that_see_zeros_first_or_nothing_else(ops, kind, scale, window, sinks):
    n_heads, heads, dim = 4, 2, 64
    spans = [(0, 100), (200, 60), (0, 50)]
    cache = R.Cache([100, 260, 50], heads, dim, 16, seed=3)
    for r, blocks in enumerate(([0, 1, 2], list(range(0, 14)), [0, 1, 2, 3])):
        for i in blocks:
            cache.vs[int(cache.table[r, i])] = 0.0
    q = (normal(5, 210, n_heads * dim) * 4).bfloat16().cuda()
    check(ops, kind, cache, spans, q, n_heads, scale, window, normal(2, n_heads) if sinks else None)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("small", [1e-6, 1e-8])
def test_zeros_among_scales_of_two_sizes(ops, kind, small):
    """Blocks of large values that few keys look at, blocks of small ones, and one of zeros."""
    n_heads, heads, dim = 4, 2, 64
    spans = [(640, 128)]
    cache = R.Cache([768], heads, dim, 16, seed=9)
    for i in range(0, 48):
        cache.vs[int(cache.table[0, i])] *= 1e-6 if i % 2 else small
    cache.vs[int(cache.table[0, 5])] = 0.0
    q = (normal(6, 128, n_heads * dim) * 1.5).bfloat16().cuda()
    check(ops, kind, cache, spans, q, n_heads, 0.25)


TAIL_KINDS = KINDS


@pytest.mark.parametrize("kind", TAIL_KINDS)
@pytest.mark.parametrize("t", [20.0, 22.3, 24.6, 25.1, 26.0])
def test_one_key_with_nearly_all_the_weight(ops, kind, t):
    """131072 positions, the first with nearly all of the weight and a value of 0, the others with 2**-t of its weight each and values: the
    output is theirs alone.  A weight is rounded to fp16 with at most 2**-32 of the largest lost (2**(t - 32) of itself), the output to
    bfloat16 (2**-9), the sum of 131072 terms in float32 by less than 2**-10."""
    n, dim, page, n_heads = 131072, 16, 128, 2
    cache = R.Cache([n], 1, dim, page, seed=1, filled=False)
    q = torch.ones(64, n_heads * dim).bfloat16()
    scale, first = 0.25, int(cache.table[0, 0])
    cache.k8[first, 0, 0] = 127
    cache.ks.fill_(t * 0.6931471805599453 / (scale * dim * 127))
    cache.v8.fill_(100)
    cache.v8[first, 0, 0] = 0
    cache.vs.fill_(0.01)
    top = scale * dim * 127 * float(cache.ks[first, 0, 0])          # the score of the first key; that of the others is 0
    last = torch.arange(n - 64, n).double()
    want = 100 * float(cache.vs[0, 0, 0]) * last * math.exp(-top) / (1 + last * math.exp(-top))
    q, spans = q.cuda(), [(n - 64, 64)]
    pos, req = R.steps(spans)
    if kind == "portions":
        out, status = portions_call(ops, cache, q, tiles_of(spans), n_heads, scale)
    else:
        out, status = rows_call(ops, cache, q if kind == "rows" else q.float(), pos, req, n_heads, scale)
    assert int(status.item()) == 0
    err = ((out.double().cpu() - want[:, None]).abs() / want[:, None]).max()
    assert float(err) <= 2.0 ** (t - 32) + 2.0 ** -9 + 2.0 ** -10, float(err)


@pytest.mark.parametrize("kind", KINDS)
def test_values_at_the_lower_end(ops, kind):
    """Values of 1e-28, whose sums of weights divided by their scale pass the range of float32: no NaN, no more than the largest value."""
    n_heads, heads, dim = 4, 2, 64
    spans = [(2900, 72)]
    cache = R.Cache([2972], heads, dim, 16, seed=4)
    cache.vs *= 1e-28
    cache.vs[int(cache.table[0, 100])] = 0.0
    q = (normal(4, 72, n_heads * dim) * 0.2).bfloat16().cuda()
    pos, req = R.steps(spans)
    if kind == "portions":
        out, status = portions_call(ops, cache, q, tiles_of(spans), n_heads, 0.1)
    else:
        out, status = rows_call(ops, cache, q if kind == "rows" else q.float(), pos, req, n_heads, 0.1)
    assert int(status.item()) == 0 and float(out.float().abs().max()) <= float(cache.vs.max()) * 127 * 1.01
