"""A key/value cache in 8 bits: each operator against its plain statement in kv8_refs.py, at the sizes where it can go wrong.

Tolerances.  Without a rotation an append is a chain of single float32 roundings that the plain statement repeats: codes and scales are
equal.  With one, sine and cosine may differ in their last bits: a turned number is off by less than 2**-21 of the block's largest, so
a value is off by at most half a step and 127 * 2**-21 of one.  Attention in float32: scores of magnitude up to S carry an error of
about (8 + S) * 2**-24 of themselves, weights the same, sums of rounded terms no more: 1e-5 of the largest value for the S of these
tests (below 30).  In bfloat16 the output is rounded to 8 bits (2**-8 of itself at most, 2**-9 on average) and the weights to 11 bits or
8: 1e-2 of the largest value."""
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


def stream():
    return torch.cuda.current_stream().cuda_stream


def word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def append(ops, cache, dev, k, v, pos, req, status, **more):
    ops.kv8_append(k, v, pos.cuda(), req.cuda(), cache.table.cuda(), *dev, status, stream(), **more)


# spans: (first position, tokens) of each request
SPANS = [[(0, 1)], [(15, 1)], [(5, 11)], [(5, 12)], [(0, 16), (0, 17), (31, 2)], [(3, 61), (16, 16), (47, 1), (0, 5)],
         [(100, 1), (7, 1), (0, 1), (15, 1), (16, 1)], [(9, 150), (0, 33)]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("spans", SPANS)
@pytest.mark.parametrize("heads,dim,dk,dv,page", [(3, 64, 64, 64, 16), (2, 48, 40, 33, 32), (1, 128, 128, 128, 64), (5, 16, 16, 16, 16),
                                                  (1, 256, 250, 256, 16), (2, 96, 96, 80, 128)])
def test_append_without_rotation_is_exact(ops, dtype, spans, heads, dim, dk, dv, page):
    cache = R.Cache([a + n for a, n in spans], heads, dim, page, seed=dim + len(spans))
    pos, req = R.steps(spans)
    T = pos.numel()
    # columns of one projection: rows at a stride of their own, keys from column 3 on (no 8-byte alignment)
    proj = (normal(T, T, 3 + heads * (dk + dv) + 2) * torch.rand(T, 1)).to(dtype).cuda()
    k, v = proj[:, 3:3 + heads * dk], proj[:, 3 + heads * dk:3 + heads * (dk + dv)]
    dev, status = cache.cuda(), word()
    append(ops, cache, dev, k, v, pos, req, status)
    for x, d, pool, scale in ((k, dk, cache.k8, cache.ks), (v, dv, cache.v8, cache.vs)):
        wide = torch.zeros(T, heads, dim)
        wide[..., :d] = x.float().cpu().view(T, heads, d)
        R.enter(cache, pool, scale, wide, pos, req)
    for got, want in zip(dev, cache.tensors()):
        assert torch.equal(got.cpu(), want)
    assert int(status.item()) == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,dk,half,interleaved,mscale", [(64, 64, 32, False, 1.0), (64, 64, 16, False, 1.25), (64, 60, 13, False, 1.0),
                                                            (128, 128, 64, False, 1.0), (48, 48, 24, True, 1.0), (96, 96, 48, False, 1.0),
                                                            (128, 128, 7, True, 0.5), (256, 256, 128, False, 1.0), (16, 16, 1, False, 1.0)])
@pytest.mark.parametrize("spans", [[(0, 1), (40, 1)], [(13, 70), (0, 20)], [(100000, 40)]])
def test_append_with_rotation(ops, dtype, dim, dk, half, interleaved, mscale, spans):
    heads, group, page = 2, 3, 16
    if spans[0][0] == 100000:
        spans = [(1000 * 16 + 7, 40)]
    cache = R.Cache([a + n for a, n in spans], heads, dim, page, seed=half, filled=False)
    pos, req = R.steps(spans)
    T = pos.numel()
    k, v, q = (normal(i + T, T, n).to(dtype).cuda() for i, n in enumerate((heads * dk, heads * dim, heads * group * dk)))
    q_out = torch.full((T, heads * group * dim), 7.0, dtype=dtype, device="cuda")
    dev, status, freq = cache.cuda(), word(), R.frequencies(half)
    append(ops, cache, dev, k, v, pos, req, status, freq=freq.cuda(), interleaved=interleaved, mscale=mscale, q=q, q_out=q_out)
    assert int(status.item()) == 0
    qw = torch.zeros(T, heads * group, dim)
    qw[..., :dk] = R.turn(q.float().cpu().view(T, heads * group, dk), pos, freq, interleaved, mscale)
    step = 2.0 ** -21 if dtype == torch.float32 else 2.0 ** -8
    assert float((q_out.float().cpu().view(T, -1, dim) - qw).abs().max()) <= step * float(qw.abs().max())
    kw = torch.zeros(T, heads, dim)
    kw[..., :dk] = R.turn(k.float().cpu().view(T, heads, dk), pos, freq, interleaved, mscale)
    cache.k8, cache.v8, cache.ks, cache.vs = (t.cpu() for t in dev)
    for t in range(T):
        p, r = int(pos[t]), int(req[t])
        pg, sub = int(cache.table[r, p // page]), p % page // 16
        block = [i for i in range(T) if int(req[i]) == r and int(pos[i]) // 16 == p // 16]
        top = kw[block].abs().amax((0, 2)) / 127
        scale = cache.ks[pg, :, sub]
        assert torch.allclose(scale, top, rtol=2.0 ** -20, atol=0)
        held = cache.held(cache.k8, cache.ks, r, p, p + 1)[:, 0]
        assert bool(((held - kw[t].double()).abs() <= scale.double()[:, None] * (0.5 + 127 * 2.0 ** -21)).all())


def test_block_filled_token_by_token(ops):
    """The scale of a block ends at its largest number whatever the steps, older codes are rounded again where it grew, and what is held is
    off by half a step for each rounding."""
    heads, dim, page, n = 2, 64, 16, 37
    x = normal(3, n, heads * dim) * torch.linspace(0.2, 3.0, n)[:, None]      # ever larger: the scale grows often
    ends = []
    for cuts in ([n], [1] * n, [5, 20, 12]):
        cache = R.Cache([n], heads, dim, page, seed=1, filled=False)
        dev, status, at = cache.cuda(), word(), 0
        for c in cuts:
            pos, req = R.steps([(at, c)])
            xc = x[at:at + c].cuda()
            append(ops, cache, dev, xc, xc * 2, pos, req, status)
            for pool, scale, f in ((cache.k8, cache.ks, 1), (cache.v8, cache.vs, 2)):
                R.enter(cache, pool, scale, x[at:at + c].view(c, heads, dim) * f, pos, req)
            at += c
        for got, want in zip(dev, cache.tensors()):
            assert torch.equal(got.cpu(), want)
        ends.append(dev[2].cpu())
        held = cache.held(cache.k8, cache.ks, 0, 0, n).transpose(0, 1).reshape(n, -1)
        steps = cache.ks.max() * (0.5 if cuts == [n] else 0.5 * 16)
        assert float((held - x.double()).abs().max()) <= float(steps) * 1.001
    assert torch.equal(ends[0], ends[1]) and torch.equal(ends[0], ends[2])


def test_numbers_that_cannot_be_held(ops):
    heads, dim, page = 1, 32, 16
    x = normal(5, 20, dim)
    x[3, 4], x[3, 5], x[4, 0], x[17] = float("nan"), float("inf"), float("-inf"), 0.0
    x[16], x[18] = 0.0, 1e-33                       # a block of nothing above 2**-100
    x[19] = 0.0
    cache = R.Cache([20], heads, dim, page, seed=2)
    pos, req = R.steps([(0, 20)])
    dev, status = cache.cuda(), word()
    append(ops, cache, dev, x.cuda(), normal(6, 20, dim).cuda(), pos, req, status)
    assert int(status.item()) == ops.ST_NOT_FINITE and "not finite" in ops.describe_status(ops.ST_NOT_FINITE)
    R.enter(cache, cache.k8, cache.ks, x.view(20, 1, dim), pos, req)
    R.enter(cache, cache.v8, cache.vs, normal(6, 20, dim).view(20, 1, dim), pos, req)
    for got, want in zip(dev, cache.tensors()):
        assert torch.equal(got.cpu(), want)
    row = dev[0].cpu()[int(cache.table[0, 0]), 0]
    assert int(row[3, 4]) == 0 and int(row[3, 5]) == 127 and int(row[4, 0]) == -127
    second = int(cache.table[0, 1])
    assert float(dev[2][second, 0, 0]) == 0.0 and int(dev[0][second, 0, :4].abs().max()) == 0


def test_rows_that_are_left_out(ops):
    """Rows of no request, pages that a request does not have, positions and page ids out of range."""
    heads, dim, page = 2, 32, 16
    cache = R.Cache([40, 40], heads, dim, page, seed=4)
    cache.table[1, 1] = -1
    before = [t.clone() for t in cache.tensors()]
    pos = torch.tensor([3, 4, 20, 21, 5], dtype=torch.int32)
    req = torch.tensor([0, -1, 1, 1, -1], dtype=torch.int32)
    k = normal(1, 5, heads * dim)
    dev, status = cache.cuda(), word()
    append(ops, cache, dev, k.cuda(), k.cuda(), pos, req, status)
    assert int(status.item()) == 0                  # a page that was given back: nothing to store
    for pool, scale in ((cache.k8, cache.ks), (cache.v8, cache.vs)):
        R.enter(cache, pool, scale, k.view(5, heads, dim), pos, req)
    for got, want in zip(dev, cache.tensors()):
        assert torch.equal(got.cpu(), want)
    table = cache.table.clone()
    table[0, 0] = before[0].shape[0]
    for p, bit in ((3, ops.ST_PAGE_RANGE), (16 * table.shape[1], ops.ST_POSITION_RANGE), (-1, ops.ST_POSITION_RANGE)):
        status = word()
        kept = [t.clone() for t in dev]
        ops.kv8_append(k[:1].cuda(), k[:1].cuda(), torch.tensor([p], dtype=torch.int32).cuda(),
                       torch.zeros(1, dtype=torch.int32).cuda(), table.cuda(), *dev, status, stream())
        assert int(status.item()) == bit
        assert all(torch.equal(a, b) for a, b in zip(kept, dev))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,dim,page", [(3, 64, 16), (2, 48, 32), (1, 256, 64)])
def test_read(ops, dtype, heads, dim, page):
    cache = R.Cache([70, 33], heads, dim, page, seed=9)
    pos = torch.tensor([0, 69, 16, 32, 15, 5], dtype=torch.int32)
    req = torch.tensor([0, 0, 0, 1, 1, -1], dtype=torch.int32)
    status = word()
    wide = torch.full((6, 2 * heads * dim + 3), 5.0, dtype=dtype, device="cuda")
    k, v = wide[:, 1:1 + heads * dim], wide[:, 1 + heads * dim:1 + 2 * heads * dim]
    ops.kv8_read(pos.cuda(), req.cuda(), cache.table.cuda(), *cache.cuda(), k, v, status, stream())
    for t in range(5):
        r, p = int(req[t]), int(pos[t])
        for got, pool, scale in ((k, cache.k8, cache.ks), (v, cache.v8, cache.vs)):
            want = cache.held(pool, scale, r, p, p + 1)[:, 0].float().to(dtype).reshape(-1)
            assert torch.equal(got[t].cpu(), want)
    assert float((wide[5].float() - 5.0).abs().max()) == 0.0 and float((wide[:, 0].float() - 5.0).abs().max()) == 0.0
    assert int(status.item()) == 0
    table = cache.table.clone()
    table[0, 0] = -1
    ops.kv8_read(pos[:1].cuda(), req[:1].cuda(), table.cuda(), *cache.cuda(), k[:1], v[:1], status, stream())
    assert int(status.item()) == ops.ST_POSITION_RANGE and float(k[0].float().abs().max()) == 0.0


def rows_call(ops, cache, q, pos, req, n_heads, scale, window=0, sinks=None, rows=None, max_len=None, status=None, table=None, out=None):
    T, dim = q.shape[0], cache.dim
    max_len = max_len or int(pos.max()) + 1
    n = T if rows is None else rows.numel()
    floats, tickets = ops.kv8_rows_scratch(n, n_heads, cache.heads, dim, max_len)
    scratch = torch.full((floats,), float("nan"), device="cuda")
    counters = torch.zeros(tickets, dtype=torch.int32, device="cuda")
    status = word() if status is None else status
    if out is None:
        out = torch.full((T, n_heads * dim), 9.0, dtype=q.dtype, device="cuda")
    table = cache.table if table is None else table
    dev = cache.cuda()
    for _ in range(2):                              # twice: the counters are left zero
        ops.kv8_attention_rows(q, pos.cuda(), req.cuda(), table.cuda(), *dev, out, n_heads, scale, window, scratch, counters, max_len,
                               status, stream(), rows=None if rows is None else rows.cuda(),
                               sinks=None if sinks is None else sinks.cuda())
    assert int(counters.abs().max()) == 0
    return out, status


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_heads,heads,dim,page", [(2, 2, 64, 16), (4, 1, 128, 16), (6, 3, 48, 32), (8, 1, 64, 16), (9, 1, 32, 64),
                                                    (1, 1, 16, 16), (5, 5, 80, 16), (16, 1, 96, 128), (3, 3, 256, 16), (10, 2, 112, 16)])
@pytest.mark.parametrize("window,with_sinks", [(0, False), (37, True)])
def test_rows(ops, dtype, n_heads, heads, dim, page, window, with_sinks):
    lengths = [1, 2, 15, 16, 17, 33, 127, 128, 129, 300, 1100]
    cache = R.Cache(lengths, heads, dim, page, seed=dim + n_heads)
    pos = torch.tensor([n - 1 for n in lengths] + [0], dtype=torch.int32)
    req = torch.tensor(list(range(len(lengths))) + [-1], dtype=torch.int32)
    T = pos.numel()
    wide = normal(dim, T, n_heads * dim + 5).to(dtype).cuda()
    q = wide[:, :n_heads * dim]                     # rows at a stride of their own
    sinks = normal(1, n_heads) if with_sinks else None
    scale = 1.5 * dim ** -0.5
    out, status = rows_call(ops, cache, q, pos, req, n_heads, scale, window, sinks)
    want = R.attention(cache, q.cpu(), pos, req, n_heads, scale, window, sinks)
    assert int(status.item()) == 0
    top = float((cache.vs.max() * 127))
    tol = 1e-5 if dtype == torch.float32 else 1e-2
    err = (out[:-1].double().cpu() - want[:-1]).abs().amax(1)
    assert float(err.max()) <= tol * top, err
    assert float((out[-1].float() - 9.0).abs().max()) == 0.0         # a row of no request


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_do_not_depend_on_their_neighbours(ops, dtype):
    lengths = [700, 20, 5000, 1300, 64]
    n_heads, heads, dim = 8, 2, 64
    cache = R.Cache(lengths, heads, dim, 16, seed=3)
    pos = torch.tensor([n - 1 for n in lengths], dtype=torch.int32)
    req = torch.arange(5, dtype=torch.int32)
    q = normal(8, 5, n_heads * dim).to(dtype).cuda()
    out, _ = rows_call(ops, cache, q, pos, req, n_heads, 0.125, max_len=8192)
    for i in range(5):
        one, _ = rows_call(ops, cache, q[i:i + 1], pos[i:i + 1], req[i:i + 1], n_heads, 0.125, max_len=8192)
        assert torch.equal(one[0], out[i])
    rows = torch.tensor([4, 1], dtype=torch.int32)
    some, _ = rows_call(ops, cache, q, pos, req, n_heads, 0.125, max_len=8192, rows=rows)
    assert torch.equal(some[4], out[4]) and torch.equal(some[1], out[1])
    assert float((some[0].float() - 9.0).abs().max()) == 0.0


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_with_large_scores_zero_scales_and_negative_scale(ops, dtype):
    lengths = [260, 40]
    n_heads, heads, dim = 4, 2, 64
    cache = R.Cache(lengths, heads, dim, 16, seed=6)
    cache.vs[int(cache.table[0, 2])] = 0.0           # a block of values of nothing
    cache.ks[int(cache.table[0, 3])] = 0.0
    cache.vs[int(cache.table[0, 4])] *= 1e4          # and one of very large ones
    pos = torch.tensor([259, 39], dtype=torch.int32)
    req = torch.arange(2, dtype=torch.int32)
    q = (normal(8, 2, n_heads * dim) * 4).to(dtype).cuda()
    for scale in (0.6, -0.6):
        out, _ = rows_call(ops, cache, q, pos, req, n_heads, scale)
        want = R.attention(cache, q.cpu(), pos, req, n_heads, scale)
        for r in range(2):
            top = max(float(want[r].abs().max()), 1e-3)
            # scores reach 0.6 * 256 * 1.2: twelve times those the bound above is for
            assert float((out[r].double().cpu() - want[r]).abs().max()) <= (1.2e-4 if dtype == torch.float32 else 2e-2) * top


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_out_of_range(ops, dtype):
    lengths = [40, 40, 40]
    n_heads, heads, dim = 2, 2, 32
    cache = R.Cache(lengths, heads, dim, 16, seed=6)
    q = normal(8, 3, n_heads * dim).to(dtype).cuda()
    req = torch.arange(3, dtype=torch.int32)
    # a position beyond the block table: the row is left as it is
    pos = torch.tensor([39, 16 * cache.table.shape[1], -5], dtype=torch.int32)
    out, status = rows_call(ops, cache, q, pos, req, n_heads, 0.2, max_len=64)
    assert int(status.item()) == ops.ST_POSITION_RANGE
    assert float((out[1:].float() - 9.0).abs().max()) == 0.0
    # a key without a page is left out of the sums, an id outside the pool too
    pos = torch.tensor([39, 39, 39], dtype=torch.int32)
    for bad, bit in ((-1, ops.ST_POSITION_RANGE), (cache.k8.shape[0], ops.ST_PAGE_RANGE)):
        table = cache.table.clone()
        table[0, 1] = bad
        out, status = rows_call(ops, cache, q, pos, req, n_heads, 0.2, table=table)
        assert int(status.item()) == bit
        k, v = cache.held(cache.k8, cache.ks, 0, 0, 40), cache.held(cache.v8, cache.vs, 0, 0, 40)
        keep = [j for j in range(40) if not 16 <= j < 32]
        s = torch.einsum("hd,hnd->hn", q[0].double().cpu().view(2, dim), k[:, keep]) * 0.2
        want = torch.einsum("hn,hnd->hd", torch.softmax(s, 1), v[:, keep]).reshape(-1)
        tol = (1e-5 if dtype == torch.float32 else 1e-2) * float(cache.vs.max() * 127)
        assert float((out[0].double().cpu() - want).abs().max()) <= tol


def tiles_of(spans):
    """Tiles of up to 128 queries for requests that bring ``[(first position, tokens)]``, rows one behind the other."""
    out, row = [], 0
    for r, (a, n) in enumerate(spans):
        out += [(row + i, min(128, n - i), r, a + i) for i in range(0, n, 128)]
        row += n
    return torch.tensor(out, dtype=torch.int32).view(-1, 4)


def portions_call(ops, cache, q, tiles, n_heads, scale, window=0, sinks=None, table=None, n_tiles=None):
    status = word()
    out = torch.full(q.shape, 9.0, dtype=q.dtype, device="cuda")
    ops.kv8_attention_portions(q, tiles.cuda(), tiles.shape[0] if n_tiles is None else n_tiles, (cache.table if table is None else table).cuda(),
                               *cache.cuda(), out, n_heads, scale, window, status, stream(), sinks=None if sinks is None else sinks.cuda())
    return out, status


PORTION_SPANS = [[(0, 1)], [(0, 128)], [(130, 7)], [(3, 129), (0, 17)], [(600, 40), (250, 140)]]


@pytest.mark.parametrize("spans", PORTION_SPANS)
@pytest.mark.parametrize("n_heads,heads,dim,page", [(2, 2, 64, 16), (4, 2, 64, 16), (4, 1, 128, 32), (3, 3, 128, 16), (6, 3, 48, 128), (5, 1, 96, 16),
                                                    (2, 1, 16, 16), (2, 2, 80, 64), (8, 2, 112, 16)])
@pytest.mark.parametrize("window,with_sinks", [(0, False), (45, True), (300, False)])
def test_portions(ops, spans, n_heads, heads, dim, page, window, with_sinks):
    cache = R.Cache([a + n for a, n in spans], heads, dim, page, seed=dim + n_heads)
    pos, req = R.steps(spans)
    T = pos.numel()
    wide = normal(dim + T, T, n_heads * dim + 3).bfloat16().cuda()
    q = wide[:, 1:1 + n_heads * dim] if page == 16 else wide[:, :n_heads * dim].contiguous()      # also rows without alignment
    sinks = normal(1, n_heads) if with_sinks else None
    scale = 1.5 * dim ** -0.5
    out, status = portions_call(ops, cache, q, tiles_of(spans), n_heads, scale, window, sinks)
    want = R.attention(cache, q.cpu(), pos, req, n_heads, scale, window, sinks)
    assert int(status.item()) == 0
    err = (out.double().cpu() - want).abs()
    assert float(err.max()) <= 1e-2 * float(cache.vs.max() * 127), float(err.max())


@pytest.mark.parametrize("n_heads,heads,dim,page", [(4, 2, 64, 16), (4, 1, 128, 32), (6, 3, 48, 128), (2, 1, 16, 16), (8, 2, 112, 16)])
@pytest.mark.parametrize("window,with_sinks", [(0, False), (45, True), (300, False)])
def test_portions_do_not_depend_on_how_many_there_are(ops, n_heads, heads, dim, page, window, with_sinks):
    """Where there are many tiles a block takes two heads, where there are few one: the same bits."""
    spans = [(3, 129), (600, 40), (0, 17), (250, 140)]
    cache = R.Cache([a + n for a, n in spans], heads, dim, page, seed=dim)
    pos, req = R.steps(spans)
    T = pos.numel()
    q = (normal(dim, T, n_heads * dim) * 2).bfloat16().cuda()
    sinks = normal(1, n_heads) if with_sinks else None
    scale = 1.5 * dim ** -0.5
    tiles = tiles_of(spans)
    few, status = portions_call(ops, cache, q, tiles, n_heads, scale, window, sinks)
    many, status2 = portions_call(ops, cache, q, torch.cat([tiles, torch.zeros(400, 4, dtype=torch.int32)]), n_heads, scale, window, sinks)
    assert int(status.item()) == 0 and int(status2.item()) == 0
    assert torch.equal(few, many)
    want = R.attention(cache, q.cpu(), pos, req, n_heads, scale, window, sinks)
    assert float((many.double().cpu() - want).abs().max()) <= 1e-2 * float(cache.vs.max() * 127)


def test_portions_with_scales_far_apart_and_released_pages(ops):
    """Blocks of nothing, blocks of very large values, pages a window has given back, tiles that pad the list, rows of no tile."""
    n_heads, heads, dim, window = 4, 2, 64, 70
    spans = [(700, 130)]
    cache = R.Cache([830], heads, dim, 16, seed=6)
    cache.vs[int(cache.table[0, 42])] = 0.0
    cache.ks[int(cache.table[0, 44])] = 0.0
    cache.vs[int(cache.table[0, 46])] *= 3e4
    cache.vs[int(cache.table[0, 47])] *= 1e-6
    pos, req = R.steps(spans)
    q = (normal(8, 140, n_heads * dim) * 3).bfloat16().cuda()
    tiles = torch.cat([tiles_of(spans), torch.zeros(2, 4, dtype=torch.int32)])
    table = cache.table.clone()
    table[0, :(700 - window + 1) // 16] = -1
    for w, t in ((window, table), (0, cache.table)):
        out, status = portions_call(ops, cache, q, tiles, n_heads, 0.3, w, table=t)
        assert int(status.item()) == 0
        want = R.attention(cache, q[:130].cpu(), pos, req, n_heads, 0.3, w).view(130, n_heads, dim)
        got = out[:130].double().cpu().view(130, n_heads, dim)
        assert float((out[130:].float() - 9.0).abs().max()) == 0.0
        top = want.abs().amax(2, keepdim=True).clamp(min=1e-3)        # each query and head by its own largest number
        assert float(((got - want).abs() / top).max()) <= 2e-2
    # a visible page that the request does not have is reported, and its keys are left out
    t = cache.table.clone()
    t[0, 45] = -1
    out, status = portions_call(ops, cache, q, tiles, n_heads, 0.3, 0, table=t)
    assert int(status.item()) == ops.ST_POSITION_RANGE
    assert bool(torch.isfinite(out[:130].float()).all())


def test_portions_and_rows_agree(ops):
    """A portion's queries one by one: the same numbers to bfloat16's precision."""
    n_heads, heads, dim = 8, 2, 128
    spans = [(1000, 150), (5, 64)]
    cache = R.Cache([1150, 69], heads, dim, 64, seed=11)
    pos, req = R.steps(spans)
    q = (normal(4, 214, n_heads * dim) * 2).bfloat16().cuda()
    out, status = portions_call(ops, cache, q, tiles_of(spans), n_heads, dim ** -0.5)
    one, _ = rows_call(ops, cache, q, pos, req, n_heads, dim ** -0.5)
    assert int(status.item()) == 0
    assert float((out.float() - one.float()).abs().max()) <= 1e-2 * float(cache.vs.max() * 127)


@pytest.mark.parametrize("pad", [0, 400])      # a head a block, two heads a block
def test_a_portion_whose_wait_runs_out(ops, pad):
    """A build with a short limit on its waits and one arrival left out (the softmax warps are never told of a tile's first scores): the
    kernel comes back by itself and says so, and the next launch of the same library, with the switch off, is right."""
    from ctypes import c_int
    from mlx_lm_b200.ops import build
    name = "kv8_portions:MLXB_TEST_WAIT_TIMEOUT=1"
    lib = build.load(name)
    lib.mlxb_test_withhold_arrival.argtypes, lib.mlxb_test_withhold_arrival.restype = [c_int], c_int
    n_heads, heads, dim = 4, 2, 128
    spans = [(500, 200)]
    cache = R.Cache([700], heads, dim, 16, seed=2)
    q = normal(3, 200, n_heads * dim).bfloat16().cuda()
    tiles = torch.cat([tiles_of(spans), torch.zeros(pad, 4, dtype=torch.int32)])
    want, _ = portions_call(ops, cache, q, tiles, n_heads, 0.1)
    real = ops._call
    try:
        ops._call = lambda lib_name, *a: real(name, *a)
        assert lib.mlxb_test_withhold_arrival(1) == 0
        out, status = portions_call(ops, cache, q, tiles, n_heads, 0.1)
        torch.cuda.synchronize()
        assert int(status.item()) == ops.ST_WAIT_TIMEOUT and bool((out == 9.0).all())
        assert lib.mlxb_test_withhold_arrival(0) == 0
        out, status = portions_call(ops, cache, q, tiles, n_heads, 0.1)
        assert int(status.item()) == 0 and torch.equal(out, want)
    finally:
        ops._call = real
        assert lib.mlxb_test_withhold_arrival(0) == 0


def test_pool_beyond_31_bits(ops):
    """Codes whose offset in the pool passes 2**31."""
    heads, dim, page = 8, 128, 128
    n_pages = 2 ** 31 // (heads * page * dim) + 3
    dev = [torch.zeros((n_pages, heads, page, dim), dtype=torch.int8, device="cuda") for _ in range(2)]
    dev += [torch.zeros((n_pages, heads, page // 16), device="cuda") for _ in range(2)]
    table = torch.tensor([[n_pages - 1, 0, n_pages - 2]], dtype=torch.int32, device="cuda")
    n = 300
    x = normal(1, n, heads * dim)
    pos, req = R.steps([(0, n)])
    status = word()
    ops.kv8_append(x.cuda(), x.cuda() * 2, pos.cuda(), req.cuda(), table, *dev, status, stream())
    small = R.Cache([n], heads, dim, page, seed=1, filled=False)
    small.table[0, :3] = torch.tensor([2, 0, 1], dtype=torch.int32)
    R.enter(small, small.k8, small.ks, x.view(n, heads, dim), pos, req)
    R.enter(small, small.v8, small.vs, x.view(n, heads, dim) * 2, pos, req)
    for a, b in ((2, n_pages - 1), (0, 0), (1, n_pages - 2)):
        for got, want in zip(dev, small.tensors()):
            assert torch.equal(got[b].cpu(), want[a])
    k, v = torch.empty(n, heads * dim, device="cuda"), torch.empty(n, heads * dim, device="cuda")
    ops.kv8_read(pos.cuda(), req.cuda(), table, *dev, k, v, status, stream())
    assert torch.equal(k.cpu(), small.held(small.k8, small.ks, 0, 0, n).float().transpose(0, 1).reshape(n, -1))
    for dtype in DTYPES:
        q = normal(2, 1, 8 * dim).to(dtype).cuda()
        floats, tickets = ops.kv8_rows_scratch(1, 8, heads, dim, 384)
        out = torch.empty_like(q)
        ops.kv8_attention_rows(q, torch.tensor([n - 1], dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda(), table, *dev, out,
                               8, dim ** -0.5, 0, torch.empty(floats, device="cuda"),
                               torch.zeros(tickets, dtype=torch.int32, device="cuda"), 384, status, stream())
        want = R.attention(small, q.cpu(), torch.tensor([n - 1]), torch.zeros(1), 8, dim ** -0.5)
        assert float((out.double().cpu() - want).abs().max()) <= (1e-5 if dtype == torch.float32 else 1e-2) * float(small.vs.max() * 127)
    assert int(status.item()) == 0


def test_on_another_stream(ops):
    """All on a stream of its own, behind work of that stream: nothing runs on the default one."""
    heads, dim, n = 2, 64, 200
    cache = R.Cache([n], heads, dim, 16, seed=1, filled=False)
    pos, req = R.steps([(0, n)])
    side = torch.cuda.Stream()
    dev, status = cache.cuda(), word()
    table, dpos, dreq = cache.table.cuda(), pos.cuda(), req.cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        x = torch.ones(n, heads * dim, device="cuda", dtype=torch.bfloat16) * 2
        ops.kv8_append(x, x, dpos, dreq, table, *dev, status, side.cuda_stream)
        out = torch.zeros(1, heads * dim, device="cuda", dtype=torch.bfloat16)
        floats, tickets = ops.kv8_rows_scratch(1, heads, heads, dim, n)
        ops.kv8_attention_rows(x[:1], dpos[-1:], dreq[-1:], table, *dev, out, heads, 0.125, 0, torch.empty(floats, device="cuda"),
                               torch.zeros(tickets, dtype=torch.int32, device="cuda"), n, status, side.cuda_stream)
    side.synchronize()
    assert float((out.float() - 2.0).abs().max()) <= 2e-2


@pytest.mark.parametrize("dtype", DTYPES)
def test_requests_rows_and_tiles_that_do_not_exist(ops, dtype):
    """A request the block table has no row for, a row of a list or of a tile beyond the queries: left out and reported."""
    n_heads, heads, dim = 4, 2, 64
    cache = R.Cache([40, 30], heads, dim, 16, seed=1)
    pos = torch.tensor([39, 5, 29], dtype=torch.int32)
    req = torch.tensor([0, 2, 1], dtype=torch.int32)         # the table has rows 0 and 1
    q = normal(2, 3, n_heads * dim).to(dtype).cuda()
    out, status = rows_call(ops, cache, q, pos, req, n_heads, 0.2)
    right, _ = rows_call(ops, cache, q, pos, torch.tensor([0, -1, 1], dtype=torch.int32), n_heads, 0.2)
    assert int(status.item()) == ops.ST_POSITION_RANGE and torch.equal(out, right)
    out, status = rows_call(ops, cache, q, pos, req, n_heads, 0.2, rows=torch.tensor([2, 3, -1, 1 << 30], dtype=torch.int32))
    assert int(status.item()) == ops.ST_POSITION_RANGE and torch.equal(out[2], right[2]) and bool((out[:2] == 9.0).all())

    dev = cache.cuda()
    before = [t.clone() for t in dev]
    x = normal(3, 3, heads * dim).to(dtype).cuda()
    s = word()
    ops.kv8_append(x, x, torch.tensor([3, 4, 5], dtype=torch.int32).cuda(), torch.tensor([2, 2, 7], dtype=torch.int32).cuda(),
                   cache.table.cuda(), *dev, s, stream())
    assert int(s.item()) == ops.ST_POSITION_RANGE and all(torch.equal(a, b) for a, b in zip(dev, before))
    s = word()
    k, v = torch.full((3, heads * dim), 9.0, dtype=dtype, device="cuda"), torch.full((3, heads * dim), 9.0, dtype=dtype, device="cuda")
    ops.kv8_read(pos.cuda(), req.cuda(), cache.table.cuda(), *dev, k, v, s, stream())
    assert int(s.item()) == ops.ST_POSITION_RANGE and not k[1].any() and not v[1].any() and k[0].any() and k[2].any()
    if dtype == torch.bfloat16:
        good = torch.tensor([(0, 2, 0, 38)], dtype=torch.int32)
        want, _ = portions_call(ops, cache, q, good, n_heads, 0.2)
        bad = torch.tensor([(2, 2, 0, 3), (-1, 1, 0, 3), (2, 1, 2, 3), (2, 1, -1, 3), (2, 1, 0, -1), (2, 1, 0, 2 ** 31 - 1)], dtype=torch.int32)
        out, status = portions_call(ops, cache, q, torch.cat([bad, good]), n_heads, 0.2)
        assert int(status.item()) == ops.ST_POSITION_RANGE and torch.equal(out, want)


def test_refusals(ops):
    cache = R.Cache([40], 2, 64, 16, seed=1)
    k8, v8, ks, vs = cache.cuda()
    table = cache.table.cuda()
    pos, req = (t.cuda() for t in R.steps([(0, 4)]))
    x = torch.zeros(4, 128, device="cuda")
    s = word()
    good = dict(k=x, v=x, positions=pos, token_req=req, block_table=table, k8=k8, v8=v8, k_scale=ks, v_scale=vs, status=s, stream=stream())
    ops.kv8_append(**good)
    bad = [dict(v=None), dict(k=x.half(), v=x.half()), dict(v=x.bfloat16()), dict(k=x[:, ::2]), dict(k=x[:, :127]), dict(v=x[:3]),
           dict(k8=k8.float()), dict(v8=v8[:, :1]), dict(k_scale=ks.half()), dict(k_scale=ks[:1]), dict(v_scale=vs.transpose(0, 1)),
           dict(block_table=table.long()), dict(block_table=table[0]), dict(positions=pos[:2]), dict(token_req=req.cpu()),
           dict(freq=torch.ones(33, device="cuda")), dict(freq=torch.ones(4, device="cuda").double()), dict(q=x), dict(q=x, q_out=x[:, :64]),
           dict(q=x[:, :120], q_out=x.clone()), dict(q=x, q_out=x), dict(k=torch.zeros(4, 144, device="cuda")),
           dict(k8=k8.view(-1, 2, 8, 64), v8=v8.view(-1, 2, 8, 64)), dict(status=s.cpu()), dict(status=s.float())]
    for change in bad:
        with pytest.raises(ops.KernelError):
            ops.kv8_append(**{**good, **change})
    read = dict(positions=pos, token_req=req, block_table=table, k8=k8, v8=v8, k_scale=ks, v_scale=vs, k_out=x.clone(), v_out=x.clone(),
                status=s, stream=stream())
    ops.kv8_read(**read)
    for change in [dict(k_out=x[:, :64]), dict(v_out=x.bfloat16()), dict(k_out=x.double(), v_out=x.double()), dict(positions=pos[:1])]:
        with pytest.raises(ops.KernelError):
            ops.kv8_read(**{**read, **change})
    floats, tickets = ops.kv8_rows_scratch(4, 4, 2, 64, 40)
    q = torch.zeros(4, 256, device="cuda")
    rows = dict(q=q, positions=pos, token_req=req, block_table=table, k8=k8, v8=v8, k_scale=ks, v_scale=vs, out=q.clone(), n_heads=4,
                scale=0.1, window=0, scratch=torch.zeros(floats, device="cuda"),
                counters=torch.zeros(tickets, dtype=torch.int32, device="cuda"), max_len=40, status=s, stream=stream())
    ops.kv8_attention_rows(**rows)
    for change in [dict(n_heads=3), dict(q=q[:, :128]), dict(out=q.bfloat16()), dict(q=q.half(), out=q.half()), dict(scratch=rows["scratch"][:-1]),
                   dict(counters=rows["counters"][:-1]), dict(positions=pos[:3]), dict(sinks=torch.zeros(3, device="cuda")),
                   dict(rows=torch.zeros(2, device="cuda")), dict(counters=rows["counters"].float()),
                   dict(rows=torch.zeros(4, dtype=torch.int32, device="cuda")[::2])]:
        with pytest.raises(ops.KernelError):
            ops.kv8_attention_rows(**{**rows, **change})
    q = q.bfloat16()
    tiles = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    portions = dict(q=q, tiles=tiles, n_tiles=2, block_table=table, k8=k8, v8=v8, k_scale=ks, v_scale=vs, out=q.clone(), n_heads=4, scale=0.1,
                    window=0, status=s, stream=stream())
    ops.kv8_attention_portions(**portions)
    for change in [dict(n_heads=3), dict(q=q.float()), dict(out=q[:2]), dict(tiles=tiles.long()), dict(n_tiles=3), dict(scale=0.0),
                   dict(scale=-1.0), dict(sinks=torch.zeros(3, device="cuda")), dict(block_table=table.long())]:
        with pytest.raises(ops.KernelError):
            ops.kv8_attention_portions(**{**portions, **change})
    assert not ops.kv8_portions_supported(torch.float32, 64) and not ops.kv8_portions_supported(torch.bfloat16, 256)
    assert int(s.item()) == 0
