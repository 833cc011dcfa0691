"""Attention over an 8-bit cache whose blocks have scales far apart, against 64 bits, each head by its own largest output.

Tolerance.  The output is rounded to bfloat16 (2**-9 of itself), a weight to fp16 (2**-12 of itself, and 2**-25 of the largest weight in all
of up to 1100 keys), the score of a key is off by 2**-16 of the scores' spread (below 100 here): 2e-3.  An output is a sum of a few weights
times codes of either sign, seldom smaller than a fifth of the largest of its head: 1e-2 of the head's largest output."""
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


KINDS = ["portions"]


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
