"""The router over more tokens than it has warps: a warp's next token is chosen for by itself, ties and near ties among them."""
import pytest
import torch

import fp8_refs as ref
from test_moe_route_plan_gpu import correction_of, logits_of, run

pytestmark = pytest.mark.gpu


def choose(logits, top, correction=None, groups=1, keep_groups=1, two=False, renormalize=False, softmax=False):
    """Choices and weights of whole tensors in 64 bits."""
    T, E = logits.shape
    z = logits.double()
    s = torch.softmax(z, -1) if softmax else torch.sigmoid(z)
    by = s + correction.double() if correction is not None else s
    if keep_groups < groups:
        per = by.view(T, groups, -1).sort(-1, descending=True).values
        judged = per[..., :2].sum(-1) if two else per[..., 0]
        kept = torch.zeros((T, groups), dtype=torch.bool, device=z.device)
        kept.scatter_(1, judged.sort(dim=-1, descending=True, stable=True).indices[:, :keep_groups], True)
        by = by.masked_fill(~kept.repeat_interleave(E // groups, 1), -torch.inf)
    sel = by.sort(dim=-1, descending=True, stable=True).indices[:, :top]
    w = s.gather(1, sel)
    return sel, w / w.sum(-1, keepdim=True) if renormalize else w


@pytest.mark.parametrize("T,E,top,groups,keep", [(8192, 256, 8, 8, 4), (5000, 256, 8, 1, 1), (6001, 64, 6, 8, 3), (5000, 500, 7, 1, 1),
                                                 (4999, 1000, 4, 8, 3)])
@pytest.mark.parametrize("softmax", [False, True])
def test_many_tokens(T, E, top, groups, keep, softmax):
    z, c = logits_of(T, E, 9), correction_of(E)
    z[::7, 5] = z[::7, 3]                        # two that would tie but for the correction
    c[3] = c[5] = 0.25
    z[3::11] = z[2]                              # the same rows again, and rows of equal numbers
    z[4::13] = 0.5
    sel, weight, order, tiles, n = run(z, top, 128, correction=c, groups=groups, keep_groups=keep, group_score="two", renormalize=True,
                                       score="softmax" if softmax else "sigmoid")
    want, w = choose(z, top, c, groups, keep, True, True, softmax)
    assert torch.equal(sel.view(T, top).long(), want)
    # float32 exponentials, a sum of at most 64 and two quotients: a few units of 2^-24 each
    assert torch.allclose(weight.view(T, top).double(), w, rtol=2e-6)
    slots, made = ref.plan(sel.tolist(), E, 128)
    assert order.tolist() == slots and int(n) == len(made) and tiles[:len(made)].tolist() == [list(t) for t in made]


@pytest.mark.parametrize("E", [60, 264])
def test_rows_that_pad_between_others(E):
    T, top = 2500, 3
    z, c = logits_of(T, E, 3), correction_of(E)
    req = torch.tensor([0 if i % 5 != 2 else -1 for i in range(T)], dtype=torch.int32, device="cuda")
    sel, weight, order, tiles, n = run(z, top, 16, req, correction=c, renormalize=True)
    want, w = choose(z, top, c, renormalize=True)
    live = (req >= 0)[:, None]
    assert torch.equal(sel.view(T, top).long(), torch.where(live, want, -1))
    assert torch.allclose(weight.view(T, top).double(), torch.where(live, w, 0.0), rtol=2e-6)
    slots, made = ref.plan(sel.tolist(), E, 16)
    assert order[:len(slots)].tolist() == slots and (order[len(slots):] == -9).all() and int(n) == len(made)
