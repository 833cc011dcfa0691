"""What an 8-bit cache holds depends on how a request was cut into steps: a block whose scale grows between two of them has its older codes
rounded again.  How far that goes.

A number is off by half a step of its block's final scale for the rounding of its own append and at most half a step for each later
append that raised the scale, so with one cut inside a block by one step.  Keys and values are then off by 1 % to 2 % of themselves on
average (a step is the block's largest number / 127, 3 to 4 times their root mean square), scores and outputs by about as much: below 5 % of the
logits (2-norm) after two or three layers, as for a cache against none."""
import pytest
import torch

from helpers import CONFIG_B, CONFIG_C, make_model_dir, random_tokens
from test_kv8_engine_gpu import load, rel, run, vocab
from lelatar_cases import CONFIG_P

pytestmark = pytest.mark.gpu


def held(engine, rid, cache=0):
    return [t.clone() for t in engine.read_cache(rid, cache)]


def cut(tokens, sizes):
    from mlx_lm_b200.engine import StepEntry
    at = 0
    for n in sizes:
        yield [StepEntry("r", tokens[at:at + n], [n - 1])]
        at += n


@pytest.mark.parametrize("sizes,roundings", [([90], 0), ([32, 48, 10], 0), ([16, 16, 16, 16, 16, 10], 0), ([23, 50, 17], 1), ([1, 89], 1), ([85, 1, 1, 1, 1, 1], 5)])
def test_what_is_held(tmp_path, sizes, roundings):
    """Layer 0 in float32, whose keys and values depend on no cache: cuts between blocks change nothing."""
    from mlx_lm_b200.engine import Engine
    model = load(tmp_path, CONFIG_B, "float32")
    tokens = random_tokens(90, vocab(CONFIG_B), 4)
    kw = dict(page_size=32, n_pages=8, max_requests=1, max_len=128)
    got = {}
    for name, bits, sz in (("full", None, [90]), ("whole", 8, [90]), ("cut", 8, sizes)):
        engine = Engine(model, kv_bits=bits, **kw)
        engine.add_request("r")
        for step in cut(tokens, sz):
            engine.step(step)
        engine.check_status()
        got[name] = held(engine, "r")
        if name == "cut":
            pages = engine.cache.requests["r"].pages[0]
            scales = [torch.stack([s[0][pages[p // 32], :, p % 32 // 16] for p in range(90)]) for s in (engine.cache.kv_groups[0].k_scale,
                                                                                                  engine.cache.kv_groups[0].v_scale)]
    for full, whole, some, scale in zip(got["full"], got["whole"], got["cut"], scales):
        if roundings == 0:
            assert torch.equal(some, whole)
        assert bool(((some - full).abs() <= scale[..., None] * 0.5 * (1 + roundings) * (1 + 2.0 ** -20)).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("config", [CONFIG_B, CONFIG_C, CONFIG_P], ids=["gpt2 B", "gpt2 C", "lelatar"])
def test_logits_of_two_budgets(tmp_path, config, dtype):
    """The same prompts under budgets of 24 and of 50 tokens a step, shared by both requests."""
    from mlx_lm_b200.engine import Engine
    model = load(tmp_path, config, dtype)
    tokens = {0: random_tokens(75, vocab(config), 1), 1: random_tokens(52, vocab(config), 2)}
    kw = dict(page_size=16, n_pages=16, max_requests=3, max_len=128, kv_bits=8)
    one = run(Engine(model, **kw), [[(0, 24)], [(0, 24)], [(0, 24)], [(0, 3), (1, 21)], [(1, 24)], [(1, 7)]], tokens)
    two = run(Engine(model, **kw), [[(0, 50)], [(0, 25), (1, 25)], [(1, 27)]], tokens)
    for r in tokens:
        assert rel(one[r], two[r]) <= 5e-2


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_request_that_was_preempted(tmp_path, dtype):
    """Tokens that came one by one come again as a portion: the logits of the next one."""
    from mlx_lm_b200.engine import Engine, StepEntry
    model = load(tmp_path, CONFIG_C, dtype)
    tokens = random_tokens(60, vocab(CONFIG_C), 7)
    engine = Engine(model, page_size=16, n_pages=8, max_requests=1, max_len=128, kv_bits=8)
    out = []
    for sizes in ([20] + [1] * 40, [60]):
        engine.add_request("r")
        for step in cut(tokens, sizes):
            last = engine.step(step).clone()
        out.append(last)
        engine.check_status()
        engine.finish("r")
    assert rel(out[0], out[1]) <= 5e-2
