"""Engines that keep keys and values in 8 bits: prompts cut in several ways, decode graphs, generation.

What is held.  Layer 0's keys and values depend on no cache, so in float32 the engine's pages are the codes that the plain statement
makes of the 32-bit engine's keys and values: equal where nothing turns, half a step off at most where the keys turn.
How far logits may be off.  A code is off by at most half a step of A / 127, A the block's largest number, 3 to 4 times its root mean
square for numbers like these: 1 % of a key or value on average.  Scores and the attention's output follow with about as much; two or
three layers of it under a residual stream stay below 5 % of the logits (2-norm)."""
import pytest
import torch

import kv8_refs as R
from helpers import CONFIG_B, CONFIG_C, make_model_dir, random_tokens
from lelatar_cases import CONFIG_P, CONFIG_S, CONFIG_T
from lelatar_cases import make_dir as make_lelatar

pytestmark = pytest.mark.gpu


def rel(a, b):
    return float((a - b).norm() / b.norm())


def load(tmp_path, config, dtype, seed=3):
    from mlx_lm_b200.weights import load_model
    if config.get("model_type") == "gpt2":
        make_model_dir(str(tmp_path), config, seed, peaky=2.0)
    else:
        make_lelatar(str(tmp_path), config, seed)
    return load_model(str(tmp_path), dtype=dtype, device="cuda:0")[0]


def vocab(config):
    return config.get("vocab_size") or config["vocab"]


def run(engine, steps, tokens):
    """Logits of every token of the requests in ``tokens``, brought in the given steps (lists of (request, tokens))."""
    from mlx_lm_b200.engine import StepEntry
    at = {r: 0 for r in tokens}
    out = {r: [] for r in tokens}
    for r in tokens:
        engine.add_request(r)
    for step in steps:
        entries = [StepEntry(r, tokens[r][at[r]:at[r] + n], list(range(n))) for r, n in step]
        logits = engine.step(entries).clone()
        for r, n in step:
            out[r].append(logits[:n])
            logits = logits[n:]
            at[r] += n
    engine.check_status()
    return {r: torch.cat(x) for r, x in out.items()}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("config", [CONFIG_B, CONFIG_C, CONFIG_P, CONFIG_S, CONFIG_T], ids=["gpt2 B", "gpt2 C", "P", "S", "T"])
@pytest.mark.parametrize("page_size", [16, 64])
def test_logits_near_those_of_the_full_cache(tmp_path, config, dtype, page_size):
    from mlx_lm_b200.engine import Engine
    model = load(tmp_path, config, dtype)
    tokens = {0: random_tokens(75, vocab(config), 1), 1: random_tokens(52, vocab(config), 2)}
    whole = [[(0, 75), (1, 52)]]
    cut = [[(0, 33)], [(0, 1), (1, 20)], [(1, 1), (0, 1)], [(0, 40), (1, 31)]]
    kw = dict(page_size=page_size, n_pages=16, max_requests=3, max_len=128)
    want = run(Engine(model, **kw), whole, tokens)
    for steps in (whole, cut):
        got = run(Engine(model, kv_bits=8, **kw), steps, tokens)
        for r in tokens:
            assert rel(got[r], want[r]) <= 5e-2
            assert bool(torch.isfinite(got[r]).all())


@pytest.mark.parametrize("config,cache", [(CONFIG_B, 0), (CONFIG_S, (1, "left"))], ids=["gpt2", "lelatar"])
def test_what_the_cache_holds(tmp_path, config, cache):
    from mlx_lm_b200.engine import Engine, StepEntry
    model = load(tmp_path, config, "float32")
    n = 41
    prompt = random_tokens(n, vocab(config), 5)
    held = {}
    for bits in (None, 8):
        engine = Engine(model, page_size=16, n_pages=8, max_requests=2, max_len=128, kv_bits=bits)
        engine.add_request("r")
        engine.step([StepEntry("r", prompt, [])])
        held[bits] = engine.read_cache("r", cache)
        engine.check_status()
        with pytest.raises(KeyError):
            engine.read_cache("r", 99)
    exact = config is CONFIG_B
    for full, got in zip(held[None], held[8]):
        full, got = full.cpu(), got.cpu()
        assert full.shape == got.shape and full.shape[0] == n
        c = R.Cache([n], full.shape[1], full.shape[2], 16, seed=1, filled=False)
        pos, req = R.steps([(0, n)])
        R.enter(c, c.k8, c.ks, full, pos, req)
        want = c.held(c.k8, c.ks, 0, 0, n).transpose(0, 1)
        if exact:
            assert torch.equal(got, want.float())
        else:      # the normed keys are rounded one by one before they turn: a code may be the neighbouring one
            step = torch.repeat_interleave(torch.stack([c.ks[int(c.table[0, i])] for i in range(3)])[..., 0], 16, 0)[:n]
            assert bool(((got - full).abs() <= step[..., None] * 0.51).all())


@pytest.mark.parametrize("config", [CONFIG_C, CONFIG_P], ids=["gpt2", "lelatar"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generation_with_and_without_graphs(tmp_path, config, dtype):
    """Greedy tokens of a batch: as decode graphs, and step by step, and each request alone in float32."""
    from mlx_lm_b200.engine import Engine
    from mlx_lm_b200.engine.scheduler import Scheduler
    from mlx_lm_b200.sampling.device import DeviceSampler
    model = load(tmp_path, config, dtype, seed=8)
    prompts = [random_tokens(n, vocab(config), n) for n in (5, 30, 17)]

    def tokens(graphs, which):
        engine = Engine(model, page_size=16, n_pages=24, max_requests=4, max_len=128, kv_bits=8)
        engine.use_graphs = graphs
        sched = Scheduler(engine, DeviceSampler(model.device, seed=0, engine=engine), max_requests=4)
        uids = [sched.insert(prompts[i], 20) for i in which]
        got = {u: [] for u in uids}
        while sched.has_work():
            for r in sched.next()[1]:
                got[r.uid].append(r.token)
        engine.check_status()
        engine.cache.check()
        return [got[u] for u in uids]

    both = tokens(True, [0, 1, 2])
    assert all(len(t) == 20 for t in both)
    assert both == tokens(False, [0, 1, 2])
    if dtype == "float32":
        assert both == [tokens(True, [i])[0] for i in range(3)]


def test_generate_and_batch_generate(tmp_path):
    from mlx_lm_b200 import batch_generate, load as load_folder, stream_generate
    make_model_dir(str(tmp_path), CONFIG_C, 3)
    model, tokenizer = load_folder(str(tmp_path))
    prompt = random_tokens(20, 640, 1)
    out = [r.token for r in stream_generate(model, tokenizer, prompt, max_tokens=8, kv_bits=8)]
    assert len(out) == 8
    r = batch_generate(model, tokenizer, [prompt, prompt[:7]], max_tokens=8, kv_bits=8, return_token_ids=True)
    assert [len(t) for t in r.token_ids] == [8, 8]
    from mlx_lm_b200.engine import Engine
    full = Engine(model, n_pages=8, max_requests=2)
    with pytest.raises(ValueError, match="kv_bits"):
        next(stream_generate(model, tokenizer, prompt, max_tokens=1, kv_bits=8, engine=full))


def test_pages_that_were_another_requests(tmp_path):
    """A page that comes back from the pool begins its blocks anew: scales of the request before do not reach the next one."""
    from mlx_lm_b200.engine import Engine, StepEntry
    model = load(tmp_path, CONFIG_C, "float32")
    engine = Engine(model, page_size=16, n_pages=4, max_requests=1, max_len=64, kv_bits=8)
    first, second = random_tokens(40, 640, 1), random_tokens(21, 640, 2)
    engine.add_request(0)
    engine.step([StepEntry(0, first, [39])])
    for g in engine.cache.kv_groups:
        g.k_scale.mul_(50.0)
    engine.finish(0)
    engine.add_request(1)
    got = engine.step([StepEntry(1, second, [20])]).clone()
    fresh = Engine(model, page_size=16, n_pages=4, max_requests=1, max_len=64, kv_bits=8)
    fresh.add_request(1)
    assert torch.equal(got, fresh.step([StepEntry(1, second, [20])]))
    # rewound into the middle of a block and brought again
    engine.cache.truncate(1, 10)
    again = engine.step([StepEntry(1, second[10:], [10])])
    assert rel(again, got) <= 5e-2
    engine.check_status()
