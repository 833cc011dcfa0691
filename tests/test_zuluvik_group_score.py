"""Zuluvik with groups judged by the sum of their two best choice scores (``router.groups.score``): the configuration reader, and the model in
float32 against the plain implementation with that rule."""
import copy
import math

import pytest
import torch

import plain_zuluvik as plain
from helpers import Trace
from lelatar_cases import run_engine, tokens, worst
from mlx_lm_b200.config import ConfigError, get_architecture
from zuluvik_cases import MOE, make_dir, model, rot, rotary


def config(score):
    mlps = [MOE(24, 10, 3, identity=2, groups=(4, 2), scale=1.5, shared=(40, 2.0)), MOE(32, 24, 4, groups=(6, 3))]
    for mlp in mlps:
        if score is not None:
            mlp["router"]["groups"]["score"] = score
    return model(120, 64, [rotary(dim=16, heads=4, kv_heads=2, vdim=16, rot_=rot(8), mlp=mlp) for mlp in mlps])


def test_the_reader():
    def experts(score):
        c = config(score)
        arch = get_architecture(c)
        return [b.feed_forward for b in arch.build(arch.args_class.from_dict(copy.deepcopy(c))).blocks]

    assert [e.group_score for e in experts("two")] == ["two", "two"]
    assert [e.group_score for e in experts(None)] == ["best", "best"] == [e.group_score for e in experts("best")]
    with pytest.raises(ConfigError, match="score"):
        experts("three")


def two_best(h, w, name, router):
    s = torch.softmax(h @ w[name + ".router"].to(h.dtype).T, dim=-1)
    choice = s + w[name + ".correction"].to(h.dtype)
    count, keep = router["groups"]["count"], router["groups"]["keep"]
    per = choice.shape[1] // count
    judged = choice.view(-1, count, per).topk(2, dim=-1).values.sum(-1)
    allowed = torch.zeros_like(judged, dtype=torch.bool).scatter_(1, judged.topk(keep, dim=-1).indices, True)
    chosen = choice.masked_fill(~allowed.repeat_interleave(per, dim=1), -math.inf).topk(router["top"], dim=-1).indices
    weight = torch.gather(s, 1, chosen)
    return weight / (weight.sum(dim=-1, keepdim=True) + 1e-20) * router["scale"], chosen


@pytest.mark.gpu
def test_the_model(tmp_path, monkeypatch):
    from mlx_lm_b200.weights import load_model

    weights = make_dir(tmp_path, config("two"), seed=3, decisive=False)
    requests = {f"r{n}": tokens(n, 120, n) for n in (1, 3, 40, 150)}
    trace = Trace()
    for rid, toks in requests.items():
        trace.whole(rid, toks)
    got = run_engine(load_model(str(tmp_path), dtype="float32")[0], trace)
    by_best = {n: plain.forward(config("two"), weights, t, dtype=torch.float64).float() for n, t in requests.items()}
    monkeypatch.setattr(plain, "route", two_best)
    by_two = {n: plain.forward(config("two"), weights, t, dtype=torch.float64).float() for n, t in requests.items()}
    assert worst(got, by_two) < 1e-5           # sums in another order, as for the other routers
    assert max(float((by_best[n] - by_two[n]).abs().max()) for n in by_two) > 1e-2       # the rule matters here
