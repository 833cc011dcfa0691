"""The bookkeeping of a cache in 8 bits, the options that ask for one, and what is refused: no GPU needed."""
import importlib

import pytest
import torch

from mlx_lm_b200 import ops
from mlx_lm_b200.cache import CacheManager
from mlx_lm_b200.config import get_architecture
from mlx_lm_b200.parts.base import PagedKVSpec, StateSpec

from helpers import CONFIG_A
from lelatar_cases import CONFIG_P
from nufetar_cases import CONFIG_A as NUFETAR


G = importlib.import_module("mlx_lm_b200.generate")      # (the package has a function of that name)


def specs_of(config):
    arch = get_architecture(config)
    return arch.build(arch.args_class.from_dict(dict(config))).cache_specs()


def test_pools_of_codes_and_scales():
    specs = {0: PagedKVSpec(2, 48, eight_bits=True), 1: PagedKVSpec(2, 48, eight_bits=True), 2: PagedKVSpec(1, 64, 100, eight_bits=True),
             3: StateSpec((3, 4))}
    m = CacheManager(specs, page_size=32, n_pages=6, max_requests=2, max_len=64, dtype=torch.bfloat16, device="cpu", kv_bits=8)
    a, b = m.kv_groups
    assert a.k.dtype == a.v.dtype == torch.int8 and a.k.shape == (2, 6, 2, 32, 48) and a.v.shape == a.k.shape
    assert a.k_scale.dtype == torch.float32 and a.k_scale.shape == a.v_scale.shape == (2, 6, 2, 2) and b.k_scale.shape == (1, 6, 1, 2)
    assert m.state_groups[0].data.shape == (1, 2, 3, 4)
    want = sum(g.k.numel() * 2 + g.k_scale.numel() * 8 for g in m.kv_groups) + 4 * m.state_groups[0].data.numel()
    assert m.nbytes() == want
    plain = CacheManager(specs, page_size=32, n_pages=6, max_requests=2, max_len=64, dtype=torch.bfloat16, device="cpu")
    assert plain.kv_groups[0].k.dtype == torch.bfloat16 and plain.kv_groups[0].k_scale is None and plain.kv_bits is None
    # pages, reservations and windows do not know of it
    m.add_request(0)
    m.reserve(0, 40)
    m.commit(0)
    m.check()
    assert m.pages_in_use() == [2, 2]


def test_which_models_can():
    for config in (CONFIG_A, CONFIG_P):
        CacheManager(specs_of(config), page_size=16, kv_bits=8)
    with pytest.raises(ValueError, match="kv_bits=8"):
        CacheManager(specs_of(NUFETAR), page_size=16, kv_bits=8)
    with pytest.raises(ValueError, match="has none"):
        CacheManager({0: StateSpec((2,))}, page_size=16, kv_bits=8)
    with pytest.raises(ValueError, match="at least 16"):
        CacheManager(specs_of(CONFIG_A), page_size=8, kv_bits=8)
    with pytest.raises(ValueError, match="kv_bits"):
        CacheManager(specs_of(CONFIG_A), page_size=16, kv_bits=4)


def test_whether_eight_bits_are_possible_does_not_tell_caches_apart():
    assert PagedKVSpec(2, 64) == PagedKVSpec(2, 64, eight_bits=True)
    assert len(CacheManager({0: PagedKVSpec(2, 64), 1: PagedKVSpec(2, 64, eight_bits=True)}).kv_groups) == 1


def test_options_and_the_engine_they_ask_for(monkeypatch):
    assert G.setup_arg_parser().parse_args(["--model", "x"]).kv_bits is None
    assert G.setup_arg_parser().parse_args(["--model", "x", "--kv-bits", "8"]).kv_bits == 8
    with pytest.raises(SystemExit):
        G.setup_arg_parser().parse_args(["--model", "x", "--kv-bits", "4"])

    class Fake:
        class cache:
            kv_bits = None

    asked = []
    monkeypatch.setattr(G, "get_engine", lambda model, **kw: asked.append(kw) or Fake)
    assert G._engine_for("m", None, 8, page_size=32) is Fake and asked == [dict(kv_bits=8, page_size=32)]
    assert G._engine_for("m", None, None) is Fake and asked[1] == {}
    assert G._engine_for("m", Fake, None) is Fake and len(asked) == 2
    with pytest.raises(ValueError, match="kv_bits"):
        G._engine_for("m", Fake, 8)


def test_what_the_kernels_take():
    assert ops.kv8_supported(16, 48) and ops.kv8_supported(128, 256)
    assert not ops.kv8_supported(8, 64) and not ops.kv8_supported(48, 64) and not ops.kv8_supported(16, 40) and not ops.kv8_supported(16, 272)
    assert ops.kv8_portions_supported(torch.bfloat16, 128) and not ops.kv8_portions_supported(torch.bfloat16, 144)
    assert not ops.kv8_portions_supported(torch.float32, 64) and not ops.kv8_portions_supported(torch.bfloat16, 64, -1.0)
    # scratch memory grows with the rows up to those of one launch, and with the longest row
    one, many = ops.kv8_rows_scratch(1, 32, 8, 128, 4096), ops.kv8_rows_scratch(64, 32, 8, 128, 4096)
    assert many == (64 * one[0], 64 * one[1])
    assert ops.kv8_rows_scratch(5000, 32, 8, 128, 4096) == ops.kv8_rows_scratch(ops.KV8_ROWS_MOST, 32, 8, 128, 4096)
    assert ops.kv8_rows_scratch(1, 16, 16, 64, 10)[0] > 0
