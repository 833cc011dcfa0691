"""Scratch memory of attention over 8-bit pages: every launch of a step works on memory that is kept, and a step whose buffers moved
while it was recorded is not issued again from that recording.  No GPU needed."""
from types import SimpleNamespace

import pytest
import torch

from mlx_lm_b200 import ops
from mlx_lm_b200.engine.step import Engine, Workspace
from mlx_lm_b200.parts import mixers


def layer(monkeypatch, ws, dtype, n_portion, n_single, tiles, head_dim=64):
    """The launches of one layer's attention: name, scratch and counters of each."""
    calls = []
    monkeypatch.setattr(ops, "kv8_attention_rows", lambda q, pos, req, table, k8, v8, ks, vs, out, n_heads, scale, window, scratch, counters,
                        max_len, status, stream, rows=None, sinks=None: calls.append(("rows", rows, scratch, counters)))
    monkeypatch.setattr(ops, "kv8_attention_portions", lambda *a, **kw: calls.append(("portions", None, None, None)))
    ctx = SimpleNamespace(ws=ws, n_portion=n_portion, n_single=n_single, portion_rows="portion rows", single_rows="single rows",
                          portion_tiles="tiles" if tiles else None, n_portion_tiles=2, positions=None, token_req=None, max_len=300,
                          status=None, stream=0)
    cache = SimpleNamespace(k=torch.zeros(2, 2, 16, head_dim, dtype=torch.int8), v=None, k_scale=torch.zeros(1), v_scale=None, block_table=None)
    mixers.paged_attention_kv8(ctx, torch.zeros(1, dtype=dtype), cache, None, 4, head_dim, 0.1, 0)
    return calls


@pytest.mark.parametrize("n_portion,n_single", [(128, 192), (192, 128), (64, 64), (0, 192), (256, 0)])
def test_launches_of_a_step_share_memory_that_is_kept(monkeypatch, n_portion, n_single):
    ws = Workspace("cpu")
    calls = [c for _ in range(2) for c in layer(monkeypatch, ws, torch.float32, n_portion, n_single, tiles=True)]
    assert [c[0] for c in calls] == ["rows"] * (2 * ((n_portion > 0) + (n_single > 0)))
    floats, tickets = ops.kv8_rows_scratch(max(n_portion, n_single), 4, 2, 64, 300)
    kept = {b.data_ptr() for b in ws._bufs.values()}
    for _, _, scratch, counters in calls:
        assert scratch.data_ptr() in kept and counters.data_ptr() in kept
        assert scratch.numel() >= floats and counters.numel() >= tickets


def test_which_launch_takes_what(monkeypatch):
    ws = Workspace("cpu")
    assert [c[:2] for c in layer(monkeypatch, ws, torch.bfloat16, 128, 64, tiles=True)] == [("portions", None), ("rows", "single rows")]
    assert [c[:2] for c in layer(monkeypatch, ws, torch.bfloat16, 128, 0, tiles=True)] == [("portions", None)]
    both = [("rows", "portion rows"), ("rows", "single rows")]
    assert [c[:2] for c in layer(monkeypatch, ws, torch.bfloat16, 128, 64, tiles=True, head_dim=256)] == both
    assert [c[:2] for c in layer(monkeypatch, ws, torch.float32, 128, 64, tiles=False)] == both


def test_a_buffer_that_moves_after_it_was_handed_out():
    ws = Workspace("cpu")
    ws.watch()
    ws.flat("a", 10, torch.float32)
    ws.flat("a", 500, torch.float32)          # (fits)
    ws.get("b", 3, 4, torch.float32)
    ws.get("c", 40, 4, torch.float32)
    assert not ws.moved
    ws.watch()
    ws.flat("a", 5000, torch.float32)         # grows at its first use: nobody has the old one
    ws.get("b", 300, 4, torch.float32)
    assert not ws.moved
    ws.get("b", 3000, 4, torch.float32)
    assert ws.moved
    ws.watch()
    ws.flat("a", 5000, torch.float32)
    assert not ws.moved
    ws.flat("a", 50000, torch.float32)
    assert ws.moved


def test_no_recording_of_a_step_whose_buffers_moved(monkeypatch):
    """A model whose second launch asks for more of the same buffer than its first."""
    monkeypatch.setattr(ops, "replay", lambda calls: ran.append("replayed"))
    ran = []

    class Model:
        def run(self, ctx):
            ran.append("ran")
            for n in sizes:
                b = engine.ws.flat("tag", n, torch.float32)
                ops._recording.append(b.data_ptr())
            return "logits"

    engine = Engine.__new__(Engine)
    engine.ws, engine.model, engine.use_replay, engine._plans, engine.n_replayed = Workspace("cpu"), Model(), True, {}, 0
    sizes = (2000, 4000)
    for want in ("ran", "ran", "replayed", "replayed"):
        assert engine._run(None, ("shape",)) == "logits"
        assert ran[-1] == want
        for gen, calls, _ in engine._plans.values():
            if gen == engine.ws.generation:
                assert set(calls) <= {b.data_ptr() for b in engine.ws._bufs.values()}
    assert engine.n_replayed == 2


def test_scratch_memory_is_bounded(monkeypatch):
    """However long the requests may be: a launch takes fewer rows then."""
    for sizes in ((32, 8, 128, 131072), (64, 8, 128, 1 << 20), (16, 16, 64, 8192), (32, 32, 256, 131072)):
        one = ops.kv8_rows_scratch(1, *sizes)
        for n in (64, 512, 5000):
            floats, tickets = ops.kv8_rows_scratch(n, *sizes)
            assert one[0] <= floats and 4 * floats <= ops.KV8_SCRATCH_MOST and floats % one[0] == 0 and tickets // one[1] == floats // one[0]
    # a buffer that grows by doubling stops at what the most rows take
    ws = Workspace("cpu")
    monkeypatch.setattr(ops, "KV8_SCRATCH_MOST", 1 << 20)
    ops._kv8_rows_at_once.cache_clear()
    try:
        for n in (40, 64, 100, 128, 512):
            layer(monkeypatch, ws, torch.float32, n, 0, tiles=False, head_dim=256)
        most = ops.kv8_rows_scratch(512, 4, 2, 256, 300)[0]
        assert max(b.numel() for b in ws._bufs.values()) == most and 4 * most <= 1 << 20
    finally:
        monkeypatch.undo()
        ops._kv8_rows_at_once.cache_clear()


def test_scratch_memory_that_is_not_all_there(monkeypatch):
    """Memory that repeats itself or lies apart has the elements and not the bytes: refused before anything is launched.  (Tensors on the
    CPU that say they are on a device; no launch gets through.)"""
    class OnDevice(torch.Tensor):
        is_cuda = True

    device = lambda t: t.as_subclass(OnDevice)
    monkeypatch.setattr(ops, "_call", lambda *a: launched.append(a[1]))
    launched = []
    codes = [device(torch.zeros(3, 2, 16, 64, dtype=torch.int8)) for _ in range(2)] + [device(torch.zeros(3, 2, 1)) for _ in range(2)]
    ints = lambda *shape: device(torch.zeros(*shape, dtype=torch.int32))
    q = device(torch.zeros(4, 256))
    floats, tickets = ops.kv8_rows_scratch(4, 4, 2, 64, 40)

    def call(scratch, counters):
        ops.kv8_attention_rows(q, ints(4), ints(4), ints(1, 3), *codes, q, 4, 0.1, 0, device(scratch), device(counters), 40, ints(1), 0)

    good = torch.zeros(floats), torch.zeros(tickets, dtype=torch.int32)
    call(*good)
    assert launched == ["mlxb_kv8_rows"]
    for bad in ((torch.zeros(1).expand(floats), good[1]), (good[0], torch.zeros(1, dtype=torch.int32).expand(tickets)),
                (torch.zeros(2 * floats)[::2], good[1]), (good[0], torch.zeros(2 * tickets, dtype=torch.int32)[::2])):
        with pytest.raises(ops.KernelError, match="contiguous"):
            call(*bad)
    assert len(launched) == 1
