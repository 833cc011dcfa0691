"""Loading a model whose weights are held in 8 bits: never more memory than what is held and a few times one block's weights in bfloat16."""
import gc

import pytest
import torch

import fisesun_cases as fisesun
from helpers import make_model_dir

pytestmark = pytest.mark.gpu

GPT2 = dict(model_type="gpt2", n_layer=16, n_embd=512, n_head=8, n_inner=2048, vocab_size=1000, n_positions=512, layer_norm_epsilon=1e-5,
            activation_function="gelu_new")
FISESUN = fisesun.model(300, 256, [fisesun.attention(dim=64, heads=4, kv_heads=2, vdim=64, v_mix=False, mlp=fisesun.MOE(512, 16, 3, shared=512))
                                   for _ in range(8)])
GPT2_BLOCK = 2 * 512 * 512 * 12
FISESUN_BLOCK = 2 * (256 * 3 * 512 * 17 + 256 * 64 * 12)


@pytest.mark.parametrize("config,make,block", [(GPT2, make_model_dir, GPT2_BLOCK), (FISESUN, fisesun.make_dir, FISESUN_BLOCK)])
def test_peak(tmp_path, config, make, block):
    """A block's weights as they arrive, as they are stacked, transposed or joined, and their codes are three times the block at most."""
    from mlx_lm_b200.weights import load_model

    make(str(tmp_path), config, 5)
    gc.collect()
    torch.cuda.empty_cache()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    model, _ = load_model(str(tmp_path), device="cuda:0", weight_bits=8)
    torch.cuda.synchronize()
    gc.collect()
    held, peak = torch.cuda.memory_allocated() - before, torch.cuda.max_memory_allocated() - before
    blocks = len(model.layers)
    assert held < 0.8 * blocks * block                  # the bfloat16 weights are gone
    assert peak <= held + 3 * block, (peak, held, block)
