"""The router of experts with its plan: choices equal to those in 64 bits, plans in one order."""
import math

import pytest
import torch

import fp8_refs as ref

pytestmark = pytest.mark.gpu


def run(logits, top, tile_rows=16, token_req=None, scratch=None, **options):
    from mlx_lm_b200 import ops

    T, E = logits.shape
    real = E - options.get("identity", 0)
    S, most = T * top, ops.moe_max_tiles(T * top, real, tile_rows)
    dev = dict(device="cuda", dtype=torch.int32)
    sel, weight = torch.full((S,), -7, **dev), torch.full((S,), -7.0, device="cuda")
    order, tiles, n = torch.full((S,), -9, **dev), torch.full((most, 3), -9, **dev), torch.full((1,), -9, **dev)
    scratch = torch.empty(ops.moe_route_scratch(T, E), **dev) if scratch is None else scratch
    ops.moe_route_plan(logits, token_req, top, sel, weight, tile_rows, order, tiles, n, scratch, ops.current_stream(), **options)
    return sel, weight, order, tiles, n


def check(logits, top, tile_rows=16, live=None, **options):
    T, E = logits.shape
    req = None if live is None else torch.tensor([0 if on else -1 for on in live], dtype=torch.int32, device="cuda")
    sel, weight, order, tiles, n = run(logits, top, tile_rows, req, **options)
    real = E - options.get("identity", 0)
    want, w = ref.route(logits.cpu(), live or [True] * T, top, score=options.get("score", "sigmoid"), correction=options.get("correction"),
                        groups=options.get("groups", 1), keep=options.get("keep_groups", 1), two=options.get("group_score") == "two",
                        renormalize=options.get("renormalize", False), eps=options.get("renormalize_eps", 0.0),
                        factor=options.get("weight_scale", 1.0), n_real=real)
    flat = [e for row in want for e in row]
    assert sel.tolist() == flat
    # float32 exponentials, a sum of at most 1024 and two quotients: a few units of 2^-24 each
    assert torch.allclose(weight.double().cpu(), torch.tensor([v for row in w for v in row], dtype=torch.float64), rtol=2e-6, atol=1e-37)
    slots, made = ref.plan(flat, real, tile_rows)
    assert int(n) == len(made)
    assert order.tolist() == slots + [-9] * (len(flat) - len(slots))
    assert tiles.tolist() == [list(t) for t in made] + [[-9] * 3] * (tiles.shape[0] - len(made))


def logits_of(T, E, seed, size=1.5):
    return (torch.randn((T, E), generator=torch.Generator().manual_seed(seed)) * size).cuda()


def correction_of(E, seed=0, size=0.05):
    return (torch.randn(E, generator=torch.Generator().manual_seed(seed)) * size).cuda()


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,top", [(1, 1), (2, 1), (8, 2), (31, 5), (33, 8), (60, 4), (64, 64), (128, 8), (160, 6), (256, 8), (500, 10), (1024, 3)])
@pytest.mark.parametrize("T", [1, 5, 64, 65, 200])
def test_choices(T, E, top, score):
    check(logits_of(T, E, T + E), top, score=score, renormalize=True, correction=correction_of(E) if T % 2 else None)


@pytest.mark.parametrize("group_score", ["best", "two"])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("corrected", [False, True])
@pytest.mark.parametrize("E,groups,keep,top", [(256, 8, 4, 8), (64, 8, 1, 3), (60, 4, 2, 4), (128, 128, 5, 5), (96, 48, 7, 8), (160, 5, 2, 6), (1000, 8, 7, 2)])
def test_groups(E, groups, keep, top, group_score, score, corrected):
    check(logits_of(97, E, E), top, tile_rows=32, score=score, groups=groups, keep_groups=keep, group_score=group_score, renormalize=True,
          correction=correction_of(E) if corrected else None, weight_scale=2.5)


@pytest.mark.parametrize("T", [3, 300])
def test_rows_that_pad_and_identities(T):
    live = [i % 3 != 1 for i in range(T)]
    check(logits_of(T, 40, 1), 6, live=live, identity=8, renormalize=True, renormalize_eps=1e-3, weight_scale=0.5, score="softmax",
          correction=correction_of(40))
    check(logits_of(T, 40, 1), 6, live=[False] * T)


@pytest.mark.parametrize("T", [40, 2000])
def test_ties_and_near_ties(T):
    """Logits out of few values, corrections that make different scores nearly equal: float32 cannot tell them apart, 64 bits can."""
    E = 64
    g = torch.Generator().manual_seed(2)
    few = (torch.randint(0, 4, (T, E), generator=g).float()).cuda()
    check(few, 7)
    check(few, 7, groups=8, keep_groups=3, group_score="two")
    z = torch.randn((T, E), generator=g)
    # a correction that brings each score to within some 1e-7 of one value
    row = torch.randn(E, generator=g)
    near = (0.6 - torch.sigmoid(row.double()) + torch.randn(E, generator=g) * 1e-7).float()
    z[::2] = row
    check(z.cuda(), 7, correction=near.cuda(), renormalize=True)
    check(z.cuda(), 7, correction=near.cuda(), groups=8, keep_groups=3, group_score="two")
    check(z.cuda(), 7, correction=near.cuda(), groups=8, keep_groups=3, group_score="best", score="softmax")


def logit(p):
    return math.log(p / (1.0 - p))


@pytest.mark.parametrize("steps", [0, 1, 3])
def test_two_that_are_close(steps):
    """Next to one of the best, at every rank and at the border of those chosen, an expert whose score is a few steps of float32 above or below."""
    T, E, top = 300, 64, 6
    z, c = logits_of(T, E, 7).cpu(), correction_of(E).cpu()
    for t in range(T):
        by = (torch.sigmoid(z[t].double()) + c.double()).sort(descending=True)
        r = t % (top + 1)
        a, b = int(by.indices[r]), int(by.indices[r + 1])
        p = float(by.values[r]) - float(c[b])
        if 0.01 < p < 0.99:
            x = torch.tensor(logit(p), dtype=torch.float32)
            for _ in range(steps):
                x = torch.nextafter(x, torch.tensor(math.inf if t % 2 else -math.inf))
            z[t, b] = x
    check(z.cuda(), top, correction=c.cuda(), renormalize=True)
    check(z.cuda(), top, correction=c.cuda(), score="softmax")


@pytest.mark.parametrize("spread", [0.0, 2e-8, 1e-7])
@pytest.mark.parametrize("n", [3, 4])
@pytest.mark.parametrize("E,top", [(64, 6), (64, 1), (256, 8), (7, 2)])
def test_several_that_are_close(E, top, n, spread):
    """Three or four scores within the rounding of float32, at every rank and on both sides of the border of those chosen."""
    T = 300
    z, c = logits_of(T, E, 9).cpu(), correction_of(E).cpu()
    g = torch.Generator().manual_seed(n)
    for t in range(T):
        by = (torch.sigmoid(z[t].double()) + c.double()).sort(descending=True)
        r = max(0, min(E - n, t % (top + 2) - 1))
        for j in range(1, n):
            b = int(by.indices[r + j])
            p = float(by.values[r]) - float(c[b]) + float(torch.randn((), generator=g)) * spread
            if 0.01 < p < 0.99:
                z[t, b] = logit(p)
    check(z.cuda(), top, correction=c.cuda(), renormalize=True)


@pytest.mark.parametrize("steps", [0, 1, 4])
@pytest.mark.parametrize("corrected", [False, True])
@pytest.mark.parametrize("E,groups,keep", [(64, 8, 3), (60, 4, 2), (96, 3, 1), (320, 5, 2)])
def test_two_groups_that_are_close(E, groups, keep, corrected, steps):
    """The last group that stays and the first that does not: sums of two a few steps of float32 apart."""
    T, per = 200, E // groups
    z, c = logits_of(T, E, 8).cpu(), correction_of(E).cpu() if corrected else torch.zeros(E)
    for t in range(T):
        by = (torch.sigmoid(z[t].double()) + c.double()).view(groups, per)
        two = by.topk(2, 1)
        order = two.values.sum(1).sort(descending=True).indices
        a, b = int(order[keep - 1]), int(order[keep])
        e = b * per + int(two.indices[b, 0])
        p = float(two.values[a].sum()) - float(two.values[b, 1]) - float(c[e])
        if 0.01 < p < 0.99:
            x = torch.tensor(logit(p), dtype=torch.float32)
            for _ in range(steps):
                x = torch.nextafter(x, torch.tensor(math.inf if t % 2 else -math.inf))
            z[t, e] = x
    check(z.cuda(), 3, correction=c.cuda() if corrected else None, groups=groups, keep_groups=keep, group_score="two")


def test_numbers_that_are_none():
    E = 40
    z = logits_of(70, E, 5)
    z[0, 3] = math.nan
    z[1] = math.nan
    z[2, :37] = math.nan
    z[3, 5] = math.inf
    z[4, 7] = -math.inf
    z[5] = -math.inf
    for T in (6, 70):
        check(z[:T], 5)
        check(z[:T], 5, groups=4, keep_groups=2, group_score="two")
        c = correction_of(E)
        c[10:20] = -math.inf
        check(z[:T], 5, correction=c, groups=4, keep_groups=2, group_score="two")
    soft = logits_of(70, E, 6)
    soft[0, 3] = math.nan
    soft[2, :37] = math.nan
    soft[4, 7] = -math.inf
    check(soft, 5, score="softmax")
    c = correction_of(E)
    c[:] = -math.inf
    c[4] = 0.0
    check(soft, 5, score="softmax", correction=c)


def test_many_tokens_and_the_same_answer_twice():
    z, c = logits_of(8192, 256, 9), correction_of(256)
    kw = dict(correction=c, groups=8, keep_groups=4, group_score="two", renormalize=True)
    first = run(z, 8, 128, **kw)
    again = run(z, 8, 128, **kw)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    sel = first[0].tolist()
    slots, made = ref.plan(sel, 256, 128)
    assert first[2].tolist() == slots and first[3][:len(made)].tolist() == [list(t) for t in made]


def test_strided_logits():
    wide = logits_of(100, 72, 3)
    check(wide[:, :60], 4)
    check(wide[:, 5:65], 4, correction=correction_of(60))


def test_agrees_with_the_router_and_the_plan_apart():
    from mlx_lm_b200 import ops

    z, top, E = logits_of(300, 64, 4), 6, 64
    sel, weight, order, tiles, n = run(z, top, 64, score="softmax", renormalize=True, groups=8, keep_groups=3)
    a, w = torch.empty_like(sel), torch.empty_like(weight)
    ops.moe_route(z, None, top, a, w, ops.current_stream(), score="softmax", renormalize=True, groups=8, keep_groups=3)
    assert torch.equal(a, sel) and torch.allclose(w, weight, rtol=1e-6)
    o, t, k = torch.empty_like(order), torch.empty_like(tiles), torch.empty_like(n)
    ops.moe_plan(sel, sel.numel(), E, 64, o, t, k, ops.current_stream())
    assert int(k) == int(n) and torch.equal(t[:int(n)], tiles[:int(n)])
    for e, first, count in tiles[:int(n)].tolist():
        assert sel[o[first:first + count].long()].tolist() == sel[order[first:first + count].long()].tolist() == [e] * count
