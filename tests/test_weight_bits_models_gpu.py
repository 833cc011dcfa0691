"""Weights in 8 bits in the architectures with side inputs, loops, recurrences and streams: against the same model with those layers computed in 64
bits from what is held, and recorded steps against themselves.

A held layer's product is off the 64-bit one's by some 7e-4 (2-norm; bfloat16 roundings of its rows flip, and roundings to 8 bits behind them); the
layers of a model add up to no more than so many times that."""
import pytest
import torch

import lelatar_cases as lelatar
import nufetar_cases as nufetar
import vobusun_cases as vobusun
from helpers import random_tokens
from test_weight_bits_gpu import CUT, WHOLE, engine, in_64_bits, rel, run     # noqa: F401

pytestmark = pytest.mark.gpu

MODELS = dict(lelatar_s=(lelatar.CONFIG_S, lelatar), lelatar_t=(lelatar.CONFIG_T, lelatar), nufetar_w=(nufetar.CONFIG_W, nufetar),
              vobusun_w=(vobusun.CONFIG_W, vobusun))


def load(path, name, **kw):
    from mlx_lm_b200.weights import load_model

    config, cases = MODELS[name]
    cases.make_dir(str(path), config, 5)
    return load_model(str(path), dtype="bfloat16", device="cuda:0", **kw)[0]


def held_products(model):
    """How many products with held weights a token goes through."""
    def of(part):
        return (getattr(part, "held", None) is not None) + sum(of(c) for c in part.children())

    d = model.description
    return sum(of(d.blocks[e.block]) if hasattr(e, "block") else of(d.reentries[e.part]) for e in d.order) + of(d.head)


@pytest.mark.parametrize("name", sorted(MODELS))
def test_logits(tmp_path, name, in_64_bits):     # noqa: F811
    vocab = MODELS[name][0]["vocab"]
    tokens = {0: random_tokens(150, vocab, 1), 1: random_tokens(90, vocab, 2)}
    model = load(tmp_path, name, weight_bits=8)
    n = held_products(model)
    assert n > 0
    whole = run(engine(model), WHOLE, tokens)
    want = run(in_64_bits(engine(model)), WHOLE, tokens)
    full = run(engine(load(tmp_path, name)), WHOLE, tokens)
    assert torch.isfinite(whole).all()
    assert rel(whole, want) <= 7e-4 * n
    assert rel(whole, full) > 1e-3


@pytest.mark.parametrize("name", sorted(MODELS))
def test_recorded_steps(tmp_path, name):
    vocab = MODELS[name][0]["vocab"]
    tokens = {0: random_tokens(150, vocab, 1), 1: random_tokens(90, vocab, 2)}
    eng = engine(load(tmp_path, name, weight_bits=8))
    first = run(eng, CUT, tokens)
    for _ in range(2):
        assert torch.equal(run(eng, CUT, tokens), first)
