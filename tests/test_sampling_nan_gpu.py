"""Rows of logits that are not numbers: the sampling kernels name a token of the vocabulary and read nothing outside the row."""
import math

import numpy as np
import pytest
import torch

from test_sampling_gpu import run_sampler

pytestmark = pytest.mark.gpu

OPTIONS = [dict(temp=0.0), dict(temp=0.7), dict(temp=1.0, top_p=0.9), dict(temp=1.0, top_k=5), dict(temp=1.0, min_p=0.1, min_tokens_to_keep=3),
           dict(temp=1.0, xtc_probability=1.0, xtc_threshold=0.1)]


@pytest.mark.parametrize("V", [33, 1000, 9000, 50257])
@pytest.mark.parametrize("options", OPTIONS)
@pytest.mark.parametrize("full", [False, True])
def test_rows_without_a_number(V, options, full):
    from mlx_lm_b200.sampling import make_sampler
    mixed = np.full(V, np.nan, dtype=np.float32)
    mixed[1::2] = -np.inf
    for row in (np.full(V, np.nan), np.full(V, -np.inf), mixed):
        tok, lp, _ = run_sampler(row, make_sampler(**options), full=full)
        assert tok == 0 and math.isnan(lp)


@pytest.mark.parametrize("V", [33, 9000, 50257])
@pytest.mark.parametrize("options", OPTIONS)
def test_one_number_among_nan(V, options):
    from mlx_lm_b200.sampling import make_sampler
    row = np.full(V, np.nan)
    row[V - 2] = -3.5
    assert run_sampler(row, make_sampler(**options))[0] == V - 2


def test_other_rows_are_as_without_them():
    """Three rows, the middle one not a number, by both kernels."""
    from mlx_lm_b200 import ops
    from mlx_lm_b200.sampling import make_sampler
    V = 20000
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, V, generator=g).cuda()
    bad = x.clone()
    bad[1] = float("nan")
    words = b"".join(make_sampler(0.8).words(5, i, 7) for i in range(3))
    params = torch.tensor(np.frombuffer(words, dtype=np.int32).copy()).cuda()

    def run(logits, sliced):
        tok, lp = torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(3, device="cuda")
        ops.sample(logits, params, tok, lp, ops.current_stream(), scratch=ops.sample_scratch(3, "cuda") if sliced else None)
        return tok.tolist(), lp.tolist()

    for sliced in (False, True):
        (tok, lp), (btok, blp) = run(x, sliced), run(bad, sliced)
        assert (btok[0], btok[2], blp[0], blp[2]) == (tok[0], tok[2], lp[0], lp[2])
        assert btok[1] == 0 and math.isnan(blp[1])
