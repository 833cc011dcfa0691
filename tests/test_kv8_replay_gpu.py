"""Steps of an engine with an 8-bit cache that are issued again from their recording: the same bits as steps that are laid out anew."""
import pytest
import torch

from helpers import CONFIG_C, make_model_dir, random_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_many_single_rows_beside_a_short_portion(tmp_path, dtype):
    """In float32 portions go row by row, like single rows, on the same scratch memory; the single rows are the larger launch."""
    from mlx_lm_b200.engine import Engine, StepEntry
    from mlx_lm_b200.weights import load_model
    make_model_dir(str(tmp_path), CONFIG_C, 5, peaky=2.0)
    model = load_model(str(tmp_path), dtype=dtype, device="cuda:0")[0]
    n, steps = 192, 4

    def run(anew):
        engine = Engine(model, page_size=16, n_pages=600, max_requests=n + steps, max_len=64, kv_bits=8)
        out = []

        def step(entries):
            if anew:
                engine._plans.clear()
            out.append(engine.step(entries).clone())

        for a in range(0, n, 4):              # a few at a time, so that the scratch memory is still small when the single rows come
            for r in range(a, a + 4):
                engine.add_request(r)
            step([StepEntry(r, random_tokens(3 + r % 5, 640, r), [0]) for r in range(a, a + 4)])
        before = engine.n_replayed
        for i in range(steps):
            engine.add_request(n + i)
            step([StepEntry(r, [7 * r % 640], [0]) for r in range(n)] + [StepEntry(n + i, random_tokens(20 + i, 640, 900 + i), [19])])
        engine.check_status()
        return out, engine.n_replayed - before

    want, none = run(anew=True)
    got, replayed = run(anew=False)
    assert none == 0 and replayed >= steps - 1
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("listed", [False, True])
def test_rows_in_several_launches(monkeypatch, dtype, listed):
    """Fewer rows at once, on the same scratch memory: the same bits."""
    import kv8_refs as R
    from mlx_lm_b200 import ops
    from test_kv8_gpu import rows_call
    lengths = [700, 20, 3000, 1300, 64, 1, 2500, 90, 17]
    n_heads, heads, dim = 8, 2, 64
    cache = R.Cache(lengths, heads, dim, 16, seed=3)
    pos = torch.tensor([n - 1 for n in lengths], dtype=torch.int32)
    req = torch.arange(len(lengths), dtype=torch.int32)
    q = torch.randn(len(lengths), n_heads * dim, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    rows = torch.tensor([8, 2, 0, 6, 3, 1, 4], dtype=torch.int32) if listed else None

    def run():
        ops._kv8_rows_at_once.cache_clear()
        ops._kv8_rows_launch.cache_clear()
        before = ops.launch_count
        out, status = rows_call(ops, cache, q, pos, req, n_heads, 0.125, max_len=8192, rows=rows)
        assert int(status.item()) == 0
        return out, ops.launch_count - before

    try:
        want, few = run()
        monkeypatch.setattr(ops, "KV8_SCRATCH_MOST", 2 * 4 * ops.kv8_rows_scratch(1, n_heads, heads, dim, 8192)[0])
        got, many = run()
        assert torch.equal(got, want) and many > few
    finally:
        monkeypatch.undo()
        ops._kv8_rows_at_once.cache_clear()
        ops._kv8_rows_launch.cache_clear()
