"""The router's choice where float32 says otherwise than 64 bits: scores under a softmax whose sum is off."""
import math

import pytest
import torch

from test_moe_route_plan_gpu import run

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
