"""Parts whose weights may be held in 8 bits, on the CPU."""
import math

import pytest
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


def bound(correction, **options):
    part = ExpertsMLP("ff", 32, 16, 8, 3, correction=True, **options)
    tensors = {s.name: torch.zeros(s.shape) for s in part.all_param_specs()}
    tensors["ff.correction"] = torch.tensor(correction)
    part.bind_all(tensors, torch.float32, "cpu")


@pytest.mark.parametrize("out", [-math.inf, math.nan])
def test_a_correction_that_leaves_too_few_experts_is_refused(out):
    """A token's third choice would be nobody, and its sum a row of an earlier step."""
    low = torch.finfo(torch.float32).min
    bound([out] * 5 + [0.0] * 3)
    bound([low] * 6 + [0.0] * 2)
    bound([out, 0.0, out, out, 0.0, 0.0, 0.0, 0.0], groups=(4, 3))
    for correction, options in (([out] * 6 + [0.0] * 2, {}), ([out, 0.0, out, out, 0.0, 0.0, 0.0, out], dict(groups=(4, 2))), ([out] * 8, {})):
        with pytest.raises(ValueError, match="fewer than the 3"):
            bound(correction, **options)
