"""Models whose weights are held in 8-bit floating point, through the engine: against the same model with those layers computed in 64 bits from
what is held, against the model in bfloat16, steps cut in several ways, decode graphs, the entry points.

How far logits may be off the 64-bit layers'.  The kernels' sums differ from exact ones by some 1e-6; a rounding to bfloat16 behind one then flips
once in a thousand times, by 2^-8 of the value, and one of those to 8 bits flips once in thirty of these, by 2^-3: some 7e-4 of a layer's
output (2-norm).  Ten or twenty of them under a residual stream stay below 1 %.

Cut in other ways, a prompt's rows go through other attention kernels, whose outputs differ by roundings to bfloat16 everywhere, not once in a
thousand times: by d = 2^-9 of a value, say.  Rounded to codes that are s = 2^-3 to 2^-4 of the value apart, numbers that differ by d fall on different codes with
probability d / s and are then s apart: sqrt(d s), 1.3 %, root mean square.  The places where rows are rounded (four a layer, three layers) add up to
sqrt(12) times that, 4.5 %, at most: below 6 %.

Off the bfloat16 model's: weights and rows are off by 2^-4 of
themselves at most, 2.6 % (root mean square) each, so 4 % of each layer's product; a few layers of it stay below 25 %."""
import pytest
import torch

import dalorax_cases as dalorax
import fisesun_cases as fisesun
import fp8_refs as ref
import zuluvik_cases as zuluvik
from helpers import make_model_dir, random_tokens

pytestmark = pytest.mark.gpu

GPT2 = dict(model_type="gpt2", n_layer=3, n_embd=256, n_head=4, n_inner=640, vocab_size=1000, n_positions=512, layer_norm_epsilon=1e-5,
            activation_function="gelu_new", ln_gain_std=0.1)
FISESUN = fisesun.model(300, 160, [fisesun.attention(dim=64, heads=4, kv_heads=2, vdim=64, v_mix=False, mlp=fisesun.MOE(136, 9, 3, shared=200)),
                                   fisesun.mlstm(dim=32, heads=4, vdim=48, mlp=fisesun.FF(200)),
                                   fisesun.attention(dim=32, heads=4, kv_heads=2, vdim=40, mlp=fisesun.MOE(264, 40, 8))])
ZULUVIK = zuluvik.model(300, 144, [zuluvik.rotary(dim=32, heads=4, kv_heads=2, vdim=48, rot_=zuluvik.rot(24, 5000.0),
                                                  mlp=zuluvik.MOE(130, 10, 3, identity=2, groups=(3, 2), scale=1.5, shared=(140, 2.0))),
                                   zuluvik.two_maps(dim=32, heads=4, kv_heads=2, vdim=40, mlp=zuluvik.MOE(200, 24, 4, scale=0.8))])
DALORAX = dalorax.model(300, 176, [dalorax.attention(dim=32, heads=6, kv_heads=2, vdim=32, mlp=dalorax.DENSE(200)),
                                   dalorax.attention(dim=32, heads=6, kv_heads=2, vdim=32, mlp=dalorax.MOE(152, 12, 2))])
MODELS = dict(gpt2=(GPT2, make_model_dir), fisesun=(FISESUN, fisesun.make_dir), zuluvik=(ZULUVIK, zuluvik.make_dir), dalorax=(DALORAX, dalorax.make_dir))


def load(path, name, **kw):
    from mlx_lm_b200.weights import load_model

    config, make = MODELS[name]
    make(str(path), config, 5)
    return load_model(str(path), dtype="bfloat16", device="cuda:0", **kw)[0]


def vocab(name):
    config = MODELS[name][0]
    return config.get("vocab_size") or config["vocab"]


def engine(model, **kw):
    from mlx_lm_b200.engine import Engine

    return Engine(model, page_size=16, n_pages=64, max_requests=8, max_len=256, **kw)


def run(eng, steps, tokens):
    from mlx_lm_b200.engine import StepEntry

    at, out = {r: 0 for r in tokens}, {r: [] for r in tokens}
    for r in tokens:
        eng.add_request(r)
    for step in steps:
        logits = eng.step([StepEntry(r, tokens[r][at[r]:at[r] + n], list(range(n))) for r, n in step]).clone()
        for r, n in step:
            out[r].append(logits[:n])
            logits = logits[n:]
            at[r] += n
    eng.check_status()
    for r in tokens:
        eng.finish(r)
    return torch.cat([torch.cat(out[r]) for r in tokens])


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.fixture
def in_64_bits(monkeypatch):
    """Layers that hold their weights in 8 bits, computed in 64 bits from what is held."""
    from mlx_lm_b200.parts.feed_forward import ExpertsMLP
    from mlx_lm_b200.parts.linear import ACTIVATIONS, Linear

    names = {code: name or "none" for name, code in ACTIVATIONS.items()}

    def linear(self, ctx, x, out, epi, residual):
        y = ref.values(x) @ ref.numbers(*self.held, self.n_in, self.n_out).T
        if self.bias is not None:
            y = y + self.bias.double()
        y = ref.ACTS[names[epi]](y)
        out.copy_(y if residual is None else y + residual.double())
        return out

    def experts(self, ctx, x, y, sel_w, plan, unit):
        order, tiles, n_tiles, _, _ = plan
        E, F, D = self.n_experts, self.inner, self.width
        w_in, w_out = ref.numbers(*self.held[0], D, F).view(E, 2, F, D), ref.numbers(*self.held[1], F, D).view(E, D, F)
        xv = ref.values(x)
        for e, first, n in tiles.view(-1, 3)[:int(n_tiles[0])].tolist():
            slots = order[first:first + n].long()
            rows = xv[slots // self.top]
            w = sel_w[slots].double()[:, None] if sel_w is not None else torch.ones(n, 1, dtype=torch.float64, device=x.device)
            h = ref.values(ref.unit(unit["unit"], rows @ w_in[e, 0].T, rows @ w_in[e, 1].T, w, unit["limit"]).float())
            y[slots] = (h @ w_out[e].T).to(y.dtype)
        return y

    def switch(eng):
        monkeypatch.setattr(Linear, "_forward_eight_bits", linear)
        monkeypatch.setattr(ExpertsMLP, "_experts_eight_bits", experts)
        eng.use_replay = eng.use_graphs = False
        return eng

    return switch


WHOLE = [[(0, 150), (1, 90)]]
CUT = [[(0, 33)], [(0, 1), (1, 20)], [(1, 1), (0, 1)], [(0, 90), (1, 69)], [(0, 25)]]


@pytest.mark.parametrize("name", sorted(MODELS))
def test_logits(tmp_path, name, in_64_bits):
    tokens = {0: random_tokens(150, vocab(name), 1), 1: random_tokens(90, vocab(name), 2)}
    model = load(tmp_path, name, weight_bits=8)
    assert model.weight_bits == 8
    whole, cut = run(engine(model), WHOLE, tokens), run(engine(model), CUT, tokens)
    full = run(engine(load(tmp_path, name)), WHOLE, tokens)
    want = run(in_64_bits(engine(model)), WHOLE, tokens)
    assert torch.isfinite(whole).all()
    assert rel(whole, want) <= 1e-2
    assert rel(cut, want) <= 6e-2
    assert 1e-3 < rel(whole, full) <= 0.25


@pytest.mark.parametrize("name", ["gpt2", "fisesun"])
def test_recorded_steps_and_graphs(tmp_path, name):
    """The same steps again, from recordings, beside other requests: the same bits."""
    model = load(tmp_path, name, weight_bits=8)
    eng = engine(model)
    tokens = {0: random_tokens(150, vocab(name), 1), 1: random_tokens(90, vocab(name), 2)}
    first = run(eng, CUT, tokens)
    for _ in range(2):
        assert torch.equal(run(eng, CUT, tokens), first)


@pytest.mark.parametrize("name", ["gpt2", "dalorax"])
def test_generation(tmp_path, name):
    """Greedy tokens of a stream (decode graphs) are those of single steps; a batch's requests end."""
    from mlx_lm_b200 import batch_generate, load as load_all, stream_generate
    from mlx_lm_b200.engine import StepEntry

    config, make = MODELS[name]
    make(str(tmp_path), config, 5)
    model, tokenizer = load_all(str(tmp_path), weight_bits=8)
    tokenizer.eos_token_ids = set()
    prompt = random_tokens(40, vocab(name), 3)
    got = [r.token for r in stream_generate(model, tokenizer, prompt, max_tokens=20)]
    eng = engine(model)
    eng.add_request(0)
    want, feed = [], prompt
    for _ in range(20):
        feed = [int(eng.step([StepEntry(0, feed, [len(feed) - 1])])[0].argmax())]
        want += feed
    assert got[:20] == want
    out = batch_generate(model, tokenizer, [prompt[:n] for n in (40, 7, 23)], max_tokens=9)
    assert len(out.texts) == 3


def test_with_a_cache_in_8_bits(tmp_path):
    model = load(tmp_path, "gpt2", weight_bits=8)
    tokens = {0: random_tokens(150, vocab("gpt2"), 1), 1: random_tokens(90, vocab("gpt2"), 2)}
    assert rel(run(engine(model, kv_bits=8), WHOLE, tokens), run(engine(model), WHOLE, tokens)) <= 5e-2


def test_memory(tmp_path):
    """What takes the weights' place is a little more than half of them, and they are gone."""
    import gc

    def held(**kw):
        gc.collect()
        torch.cuda.empty_cache()
        before = torch.cuda.memory_allocated()
        model = load(tmp_path, "gpt2", **kw)
        gc.collect()
        return torch.cuda.memory_allocated() - before, model

    full, a = held()
    eight, b = held(weight_bits=8)
    layers = 3 * 2 * (256 * 768 + 256 * 256 + 2 * 256 * 640)
    assert full - eight >= 0.4 * layers
    assert all(l.weight is None and l.held is not None for block in b.layers for l in (block.mixer.qkv, block.feed_forward.up, block.feed_forward.down))


def test_float32_is_refused(tmp_path):
    from mlx_lm_b200.weights import load_model

    make_model_dir(str(tmp_path), GPT2, 5)
    with pytest.raises(ValueError, match="weight_bits=8"):
        load_model(str(tmp_path), dtype="float32", device="cuda:0", weight_bits=8)
    with pytest.raises(ValueError, match="weight_bits"):
        load_model(str(tmp_path), device="cuda:0", weight_bits=4)


def test_a_model_without_such_weights_is_refused(tmp_path):
    from mlx_lm_b200.weights import load_model

    make_model_dir(str(tmp_path), dict(GPT2, n_embd=64, n_inner=96), 5)
    with pytest.raises(ValueError, match="no weight"):
        load_model(str(tmp_path), device="cuda:0", weight_bits=8)


# ------------------------------------------------------------------------------------------------ groups judged by two

@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, None), (torch.float32, None), (torch.bfloat16, 8)])
@pytest.mark.parametrize("T", [3, 200])
def test_experts_in_groups_judged_by_two(dtype, bits, T):
    """A feed-forward of experts with such a router in bfloat16, float32 and 8 bits, its parts by hand."""
    from types import SimpleNamespace

    from mlx_lm_b200 import ops
    from mlx_lm_b200.engine.step import Workspace
    from mlx_lm_b200.parts.feed_forward import ExpertsMLP

    D, F, E, top = 160, 136, 16, 3
    part = ExpertsMLP("ff", D, F, E, top, score="sigmoid", renormalize=True, correction=True, groups=(4, 2), group_score="two", weight_scale=1.5)
    part.set_weight_bits(bits)
    g = torch.Generator().manual_seed(T)
    tensors = {s.name: (torch.randn(s.shape, generator=g) * (0.05 if "correction" in s.name else s.shape[-1] ** -0.5)).cuda() for s in part.all_param_specs()}
    part.bind_all({n: t if "correction" in n else t.to(dtype) for n, t in tensors.items()}, dtype, "cuda")
    if bits:
        assert part.hold_eight_bits() == 1 and part.w_in is None and part.router.weight is not None
    x = torch.randn((T, D), generator=g).to(dtype).cuda()
    req = torch.zeros(T, dtype=torch.int32, device="cuda")
    req[1] = -1
    ctx = SimpleNamespace(ws=Workspace("cuda"), stream=ops.current_stream(), token_req=req, status=torch.zeros(1, dtype=torch.int32, device="cuda"),
                          n_tokens=T, leading_portion_rows=0, dtype=dtype)
    y, sel, weight = part._experts(ctx, x)
    torch.cuda.synchronize()
    assert int(ctx.status) == 0
    logits = ctx.ws.get("moe_logits", T, E, torch.float32)[:, :E]
    live = [r >= 0 for r in req.tolist()]
    want, w = ref.route(logits.cpu(), live, top, correction=part.correction.cpu(), groups=4, keep=2, two=True, renormalize=True, factor=1.5)
    assert sel[:T * top].tolist() == [e for row in want for e in row]
    assert any(a != b for a, b in zip(want, ref.route(logits.cpu(), live, top, correction=part.correction.cpu(), groups=4, keep=2)[0])) or T < 10
    hold = ref.values if bits else (lambda t: t.double())
    half = (lambda t: ref.values(t)) if bits else (lambda t: t.to(dtype).double())
    for t in range(T):
        for c in range(top):
            e = want[t][c]
            if e < 0:
                continue
            names = part.names[e]
            m = [hold(tensors[n].to(dtype)) for n in names]
            row = hold(x[t:t + 1])
            h = half(ref.unit("silu", row @ m[0].T, row @ m[1].T, w[t][c], 0.0).float())
            err = (y[t * top + c].double() - (h @ m[2].T)[0]).norm() / (h @ m[2].T).norm()
            # float32: sums of 160; bfloat16: the hidden row's roundings may flip; 8 bits: so may these, by more
            assert float(err) <= (1e-5 if dtype == torch.float32 else 2e-2 if bits else 4e-3)
