"""Appends to an 8-bit cache whose rows or numbers are not what a step of an engine brings."""
import pytest
import torch

import kv8_refs as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    from mlx_lm_b200 import ops as o
    o.require_cuda()
    return o


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


# positions of a request's rows, and which of them enter
ASTRAY = [([3, 5], [3]), ([3, 4, 6, 7], [3, 4]), ([5, 5], [5]), ([20, 21, 3], [20, 21]), ([0, 2, 3, 4, 16, 17], [0, 16, 17]),
          ([3, 20, 21], [3, 20, 21]), ([14, 15, 17, 18], [14, 15, 17, 18]), ([8, 7, 6], [8]), (list(range(5, 16)) + [2, 3], list(range(5, 16)))]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ahead", [0, 15, 16, 300])      # rows of another request in front: a row a block, 16 a block, at their edges
@pytest.mark.parametrize("positions,enter", ASTRAY)
def test_rows_out_of_order_or_with_gaps(ops, dtype, ahead, positions, enter):
    heads, dim, page = 2, 64, 16
    cache = R.Cache([40, max(1, ahead)], heads, dim, page, seed=len(positions) + ahead)
    pos = torch.tensor(list(range(ahead)) + positions, dtype=torch.int32)
    req = torch.tensor([1] * ahead + [0] * len(positions), dtype=torch.int32)
    T = pos.numel()
    x = normal(T, T, heads * dim).to(dtype)
    q = normal(T + 1, T, heads * dim).to(dtype).cuda()
    q_out = torch.zeros_like(q)
    dev, status = cache.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.kv8_append(x.cuda(), x.cuda(), pos.cuda(), req.cuda(), cache.table.cuda(), *dev, status, ops.current_stream(), q=q, q_out=q_out)
    entered = torch.cat([torch.ones(ahead, dtype=torch.bool), torch.zeros(len(positions), dtype=torch.bool)])
    left = list(enter)
    for i, p in enumerate(positions):
        if left and p == left[0]:
            entered[ahead + i] = True
            left.pop(0)
    assert not left
    for pool, scale in ((cache.k8, cache.ks), (cache.v8, cache.vs)):
        R.enter(cache, pool, scale, x.float().view(T, heads, dim), pos, torch.where(entered, req, -1))
    for got, want in zip(dev, cache.tensors()):
        assert torch.equal(got.cpu(), want)
    assert int(status.item()) == (0 if len(enter) == len(positions) else ops.ST_POSITION_RANGE)
    assert torch.equal(q_out, q)                # (queries write to rows of their own: any order will do)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("aligned", [True, False])
def test_infinities_beside_the_largest_number(ops, dtype, aligned):
    """An infinity is held as the largest code of its sign whatever else its block holds, up to the type's largest number."""
    top = torch.finfo(dtype).max
    x = torch.zeros(4, 33)
    x[0, :4] = torch.tensor([top, float("inf"), float("-inf"), float("nan")])
    x[1, 1] = -top
    x[2, 0] = float("inf")
    x = x.to(dtype).cuda()
    k = x[:, :32].contiguous() if aligned else x[:, :32]
    cache = R.Cache([4], 1, 32, 16, seed=1, filled=False)
    dev, status = cache.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    pos, req = R.steps([(0, 4)])
    ops.kv8_append(k, k, pos.cuda(), req.cuda(), cache.table.cuda(), *dev, status, ops.current_stream())
    page = int(cache.table[0, 0])
    for codes, scale in ((dev[0], dev[2]), (dev[1], dev[3])):
        row = codes[page, 0].cpu()
        assert row[0, :5].tolist() == [127, 127, -127, 0, 0] and row[1, :3].tolist() == [0, -127, 0] and int(row[2, 0]) == 127
        assert float(scale[page, 0, 0]) == float(torch.tensor(top) / 127)
    assert int(status.item()) == ops.ST_NOT_FINITE
