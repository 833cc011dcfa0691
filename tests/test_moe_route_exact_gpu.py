"""The router's choice where float32 says otherwise than 64 bits: scores under a softmax whose sum is off, groups whose two best cancel."""
import math

import pytest
import torch

from test_moe_route_plan_gpu import check, correction_of, logits_of, run

pytestmark = pytest.mark.gpu


def choices(z, correction, top, **options):
    """What the kernel chooses and what 64 bits choose, in rows."""
    T, E = z.shape
    by = torch.softmax(z.double(), -1) + correction.double()
    if options:
        groups = options["groups"]
        two = by.view(T, groups, -1).sort(-1, descending=True).values[..., :2].sum(-1)
        best = two.sort(dim=-1, descending=True, stable=True).indices[:, :options["keep_groups"]]
        kept = torch.zeros((T, groups), dtype=torch.bool, device=z.device).scatter(1, best, True)
        by = by.masked_fill(~kept.repeat_interleave(E // groups, 1), -math.inf)
    return run(z, top, score="softmax", correction=correction, **options)[0].view(T, top).long(), by.sort(dim=-1, descending=True, stable=True).indices[:, :top]


@pytest.mark.parametrize("E", [64, 256, 512, 1024])
@pytest.mark.parametrize("by", [-4e-7, -1.4e-7, 1.4e-7, 4e-7])
def test_softmax_one_far_ahead(E, by):
    """Logits 0 for one expert and such for all others that a sum of their exponentials, one after the other, is rounded the same way every time;
    and others, that an error of the exponential is the same for all of them.  A correction puts expert 1 ahead of expert 0 by `by`."""
    others = [math.log((n + cut) * 2.0 ** -23) for n in (17, 63, 200) for cut in (0.42, 0.58)] + [-2.0 - 0.21 * i for i in range(30)]
    for x in others:
        z = torch.full((150, E), x)
        z[:, 0] = 0.0
        s = torch.softmax(z[0].double(), -1)
        c = torch.zeros(E)
        c[1] = float(s[0] - s[1] + by)
        for T in (1, 150):
            got, want = choices(z[:T].cuda(), c.cuda(), 1)
            assert torch.equal(got, want)


@pytest.mark.parametrize("E", [256, 1024])
@pytest.mark.parametrize("by", [-3e-7, -1e-7, 1e-7, 3e-7])
def test_softmax_groups_of_two_one_far_ahead(E, by):
    """The same where groups are chosen by the sum of their two best: a group with expert 0 and one whose best has a correction."""
    for x in [math.log((n + cut) * 2.0 ** -23) for n in (17, 63, 200) for cut in (0.42, 0.58)] + [-2.0 - 0.5 * i for i in range(12)]:
        z = torch.full((1, E), x)
        z[0, 0] = 0.0
        s = torch.softmax(z[0].double(), -1)
        c = torch.zeros(E)
        c[E // 2] = float(s[0] - s[1] + by)
        got, want = choices(z.cuda(), c.cuda(), 2, groups=4, keep_groups=1, group_score="two")
        assert torch.equal(got, want)


@pytest.mark.parametrize("size", [30.0, 1000.0, 1e5])
@pytest.mark.parametrize("groups,per", [(8, 2), (4, 3), (16, 4)])
def test_two_best_that_cancel(size, groups, per):
    """Corrections far above and far below zero in every group: sums of two are small, their float32 roundings are not."""
    T, E, keep = 200, groups * per, groups // 2
    g = torch.Generator().manual_seed(groups)
    c = torch.full((groups, per), -10.0 * size)
    c[:, 0], c[:, 1] = size, -size
    z = torch.randn((T, groups, per), generator=g)
    for t in range(T):                # the last that stays and the first that goes, nearer to one another than the size's rounding
        two = torch.sigmoid(z[t, :, :2].double()).sum(1)
        order = two.sort(descending=True).indices
        a, b = int(order[keep - 1]), int(order[keep])
        p = float(two[a]) - float(torch.sigmoid(z[t, b, 1].double())) + float(torch.randn((), generator=g)) * size * 2.0 ** -26
        if 0.01 < p < 0.99:
            z[t, b, 0] = math.log(p / (1.0 - p))
    check(z.view(T, E).cuda(), 2, correction=c.view(E).cuda(), groups=groups, keep_groups=keep, group_score="two", renormalize=True)


@pytest.mark.parametrize("corrected", ["lowest", "halves"])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_groups_out_of_the_lowest_numbers(corrected, score):
    """Groups whose corrections are the type's lowest number, or half of it: they come last, and are chosen from where nothing else is left."""
    T, groups, per = 90, 8, 4
    lowest = torch.finfo(torch.float32).min
    c = correction_of(groups * per).view(groups, per)
    c[3:] = lowest if corrected == "lowest" else 0.5 * lowest
    c[1, 2:] = lowest
    c[5, 1] = -math.inf
    for keep, top in ((2, 3), (3, 8), (5, 14)):
        for two in ("best", "two"):
            check(logits_of(T, groups * per, keep), top, correction=c.view(-1).contiguous(), groups=groups, keep_groups=keep, group_score=two, score=score)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,groups,keep", [(40, 1, 1), (64, 8, 3), (96, 48, 7), (600, 6, 2)])
def test_the_two_zeros_are_equal(E, groups, keep, score):
    """Logits of plus and minus zero among others: the lower index is chosen."""
    z = (torch.randn((130, E), generator=torch.Generator().manual_seed(E)) * 0.3).round()
    assert (torch.signbit(z) & (z == 0)).any(1).all() and (~torch.signbit(z) & (z == 0)).any(1).all()
    for two in ("best", "two"):
        check(z.cuda(), 6, score=score, groups=groups, keep_groups=keep, group_score=two)
        check(z.cuda(), 6, score=score, groups=groups, keep_groups=keep, group_score=two, correction=torch.zeros(E, device="cuda"))
