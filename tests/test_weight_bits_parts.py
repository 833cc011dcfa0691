"""Parts whose weights may be held in 8 bits, on the CPU."""
import torch

from mlx_lm_b200.parts.feed_forward import ExpertsMLP
from mlx_lm_b200.parts.linear import FusedLinear, Linear


def test_a_part_that_is_bound_again_holds_nothing_of_before():
    linear, fused, experts = Linear("l", 128, 256, bias=False), FusedLinear("f", 128, [("a", 64), ("b", 64)]), ExpertsMLP("ff", 128, 64, 4, 2)
    for part in (linear, fused, experts):
        part.set_weight_bits(8)
        part.held = (torch.zeros(1), torch.zeros(1))          # as hold_eight_bits leaves it
        part.set_weight_bits(None)
        assert part.held is None and part.weight_bits is None
        part.bind_all({s.name: torch.zeros(s.shape, dtype=torch.bfloat16) for s in part.all_param_specs()}, torch.bfloat16, "cpu")
        assert part.held is None
