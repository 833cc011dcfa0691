"""A key or value that an 8-bit cache cannot hold ends its own request and no other."""
import warnings

import pytest
import torch

import kv8_refs as R
from helpers import CONFIG_C, make_model_dir, random_tokens
from lelatar_cases import CONFIG_P
from lelatar_cases import make_dir as make_lelatar

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [3, 40])                # rows of each request; more than 256 in all: 16 rows a block
def test_flags_of_requests(dtype, rows):
    from mlx_lm_b200 import ops
    heads, dim, n = 2, 64, 9
    cache = R.Cache([rows] * n, heads, dim, 16, seed=1, filled=False)
    pos, req = R.steps([(0, rows)] * n)
    x = torch.randn(n * rows, heads * dim, generator=torch.Generator().manual_seed(2))
    y = x.clone()
    x[2 * rows, 5] = float("nan")                        # request 2: a key
    y[8 * rows - 1, 70] = float("-inf")                  # request 7: a value
    slots = torch.tensor([30, 4, 17, 2, 9, 11, 12, 25, 1], dtype=torch.int32, device="cuda")
    flags, status = torch.zeros(31, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    args = [t.to(dtype).cuda() for t in (x, y)] + [pos.cuda(), req.cuda(), cache.table.cuda(), *cache.cuda(), status, ops.current_stream()]
    ops.kv8_append(*args, not_finite=flags, slots=slots)
    assert flags.nonzero().flatten().tolist() == [17, 25] and int(flags.max()) == 1
    assert int(status.item()) == ops.ST_NOT_FINITE
    flags = torch.zeros(20, dtype=torch.int32, device="cuda")
    ops.kv8_append(*args, not_finite=flags, slots=slots)        # slot 25 is not among them: the status word alone says so
    assert flags.nonzero().flatten().tolist() == [17]
    for more in (dict(not_finite=flags), dict(slots=slots), dict(not_finite=flags, slots=slots[:8]), dict(not_finite=flags.float(), slots=slots),
                 dict(not_finite=flags, slots=slots.long()), dict(not_finite=flags.cpu(), slots=slots)):
        with pytest.raises(ops.KernelError):
            ops.kv8_append(*args, **more)


def gpt2(tmp_path, dtype, broken):
    from mlx_lm_b200.weights import load_model
    make_model_dir(str(tmp_path), CONFIG_C, 3, peaky=2.0)
    model = load_model(str(tmp_path), dtype=dtype, device="cuda:0")[0]
    if broken:
        model.description.position.table[40] = float("inf")      # whoever gets to position 40
    return model


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_batch_goes_on(tmp_path, dtype, graphs):
    from mlx_lm_b200.engine import Engine
    from mlx_lm_b200.engine.scheduler import Scheduler
    from mlx_lm_b200.sampling.device import DeviceSampler
    prompts = [random_tokens(n, 640, n) for n in (5, 45, 30, 12)]

    def tokens(broken):
        model = gpt2(tmp_path, dtype, broken)
        engine = Engine(model, page_size=16, n_pages=40, max_requests=4, max_len=128, kv_bits=8)
        engine.use_graphs = graphs
        sched = Scheduler(engine, DeviceSampler(model.device, seed=0, engine=engine), max_requests=4)
        uids = [sched.insert(p, 20) for p in prompts]
        got, why = {u: [] for u in uids}, {}
        while sched.has_work():
            for r in sched.next()[1]:
                got[r.uid].append(r.token)
                if r.finish_reason:
                    why[r.uid] = r.finish_reason
        engine.check_status()
        engine.cache.check()
        assert not engine.cache.requests and not engine.failed and not engine.not_finite.any()
        return [got[u] for u in uids], [why[u] for u in uids]

    want, _ = tokens(False)
    got, why = tokens(True)
    assert why == ["length", "not_finite", "not_finite", "length"]
    assert got[1] == [-1] and got[2][-1] == -1 and len(got[2]) == 12       # positions 30 to 39 are fed behind the first token
    assert len(got[0]) == len(got[3]) == 20
    if dtype == "float32":      # (a row's bits do not depend on who else is in the batch)
        assert got[0] == want[0] and got[3] == want[3] and got[2][:-1] == want[2][:11]


def test_a_slot_is_clean_for_its_next_request(tmp_path):
    from mlx_lm_b200 import ops
    from mlx_lm_b200.engine import Engine, StepEntry
    model = gpt2(tmp_path, "float32", True)
    engine = Engine(model, page_size=16, n_pages=8, max_requests=1, max_len=64, kv_bits=8)
    engine.add_request(0)
    engine.step([StepEntry(0, random_tokens(45, 640, 1), [44])])
    engine.finish(0)                                     # nobody has asked
    engine.add_request(1)
    engine.step([StepEntry(1, random_tokens(20, 640, 1), [19])])
    engine.find_not_finite()
    assert not engine.failed
    engine.check_status()
    engine.step([StepEntry(1, random_tokens(25, 640, 2), [24])])
    with pytest.raises(ops.KernelError, match="not finite"):
        engine.check_status()
    engine.find_not_finite()
    assert engine.failed == {1}
    engine.finish(1)
    assert not engine.failed


def test_generation(tmp_path):
    from mlx_lm_b200 import batch_generate, load, ops, stream_generate
    make_model_dir(str(tmp_path), CONFIG_C, 3)
    model, tokenizer = load(str(tmp_path))
    model.description.position.table[40] = float("inf")
    prompts = [random_tokens(n, 640, n) for n in (7, 38)]
    with pytest.warns(UserWarning, match="request 1 ended after 3 tokens"):
        r = batch_generate(model, tokenizer, prompts, max_tokens=9, kv_bits=8, return_token_ids=True, return_logprobs=True)
    assert [len(t) for t in r.token_ids] == [9, 3] and [len(t) for t in r.logprobs] == [9, 3]      # positions 38 and 39 are fed behind the first
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        again = batch_generate(model, tokenizer, prompts[:1], max_tokens=9, kv_bits=8, return_token_ids=True)
    assert len(again.token_ids[0]) == 9
    with pytest.raises(ops.KernelError, match="not finite"):
        list(stream_generate(model, tokenizer, prompts[1], max_tokens=9, kv_bits=8))
    assert len(list(stream_generate(model, tokenizer, prompts[0], max_tokens=9, kv_bits=8))) == 9


def test_layers_that_turn_their_keys_say_whose_it_was(tmp_path):
    from mlx_lm_b200.engine import Engine, StepEntry
    from mlx_lm_b200.weights import load_model
    make_lelatar(str(tmp_path), CONFIG_P, 3)
    model = load_model(str(tmp_path), dtype="bfloat16", device="cuda:0")[0]
    vocab = CONFIG_P.get("vocab_size") or CONFIG_P["vocab"]
    engine = Engine(model, page_size=16, n_pages=12, max_requests=3, max_len=64, kv_bits=8)
    for r in range(3):
        engine.add_request(r)
    good = [t % (vocab - 1) for t in random_tokens(20, vocab, 1)]
    model.description.embedding.table[vocab - 1] = float("nan")
    engine.step([StepEntry(0, good, [19]), StepEntry(1, good[:10] + [vocab - 1], [10]), StepEntry(2, good[:3], [2])])
    engine.find_not_finite()
    assert engine.failed == {1}
    engine.check_status()
