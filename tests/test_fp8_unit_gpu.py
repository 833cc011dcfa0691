"""The gated unit in front of the 8 bits: as near to 64 bits for gates far below zero as for small ones."""
import pytest
import torch

import fp8_refs as ref
from test_fp8_gpu import kept, planned, status

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tile_rows", [16, 128])
@pytest.mark.parametrize("depth", [0.0, 16.0, 40.0, 56.0])
def test_unit(tile_rows, depth):
    """Products that float32 holds exactly: rows and weights are a few codes of 4 bits at powers of two (18 bits in all).  Then the unit alone is
    rounded before the 8 bits: by 10 * 2^-24 of itself at most (exponential and quotient two units in the last place, each 2^-23; a sum and a product, each
    2^-24).  The number held must be the one that a number so near rounds to."""
    from mlx_lm_b200 import ops as o

    T, D, F = 1024, 128, 2048
    g = torch.Generator().manual_seed(int(depth))
    x = torch.zeros((T, D))
    s = (8 + torch.randint(0, 8, (T, 3), generator=g)) / 8.0
    x[:, 0], x[:, 1], x[:, 2], x[:, 3] = s[:, 0], s[:, 1] / 16, s[:, 2] / 256, 1.0
    w = torch.zeros((2 * F, D))
    w[:, :3] = torch.randint(-15, 16, (2 * F, 3), generator=g) / 8.0
    w[:F, 3] = -depth
    x, w = x.bfloat16().cuda(), w.bfloat16().cuda()
    assert torch.equal(ref.values(x), x.double()) and torch.equal(ref.values(w), w.double())
    plan = planned([0] * T, 1, tile_rows)
    codes, scales = o.fp8_empty(tile_rows, D, "cuda", groups=plan[3])
    hc, hs = o.fp8_empty(tile_rows, F, "cuda", groups=plan[3])
    st, stream = status(), o.current_stream()
    o.moe_gather_fp8(x, 1, *plan, codes, scales, stream)
    o.moe_gemm_fp8(codes, scales, *kept(w, F), *plan, hc, st, stream, gated=True, out_scales=hs)
    got = ref.numbers(hc, hs, F, tile_rows)[:T]
    gate, up = x.double() @ w[:F].double().T, x.double() @ w[F:].double().T
    h = ref.unit("silu", gate, up, 1.0, 0.0)
    near = 10.0 * 2.0 ** -24
    (lo, lo_e), (hi, hi_e) = ref.held(h * (1 - near)), ref.held(h * (1 + near))
    same = lo_e == hi_e                       # a run whose scale hangs on it is left out: its largest number is that near to 448 times a power of two
    assert float(same.double().mean()) > 0.99
    of = lambda c, e: torch.ldexp(c, e.repeat_interleave(ref.RUN, 1))
    fits = (got == of(lo, lo_e)) | (got == of(hi, hi_e)) | ~same.repeat_interleave(ref.RUN, 1)
    assert int(st) == 0 and fits.all(), (int((~fits).sum()), fits.numel())
