"""Forms of the experts' products in 8 bits: K split over a cluster, rows of results that begin anywhere, more tiles than CTAs."""
import pytest
import torch

from test_fp8_gpu import check_experts, kept, normal, planned, status

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ranks", [1, 2, 4, 8])
@pytest.mark.parametrize("unit,weighted,out_dtype", [("silu", True, torch.bfloat16), ("bounded", False, torch.float32)])
def test_experts_with_k_split(monkeypatch, ranks, unit, weighted, out_dtype):
    """Sums that the CTAs of a cluster share: odd numbers of runs, tiles of 1, 5 and 16 slots, clusters behind the plan's last tile."""
    monkeypatch.setenv("MLXB_FP8_RANKS", str(ranks))
    sel = [0] + [1] * 5 + [2] * 16 + [4] * 37 + [-1] * 5
    check_experts(32, 2, 6, 1100, 1160, 16, unit=unit, limit=2.0, weighted=weighted, out_dtype=out_dtype, sel=sel)
    check_experts(3, 2, 40, 1024, 1024, 16, unit=unit, limit=2.0, weighted=weighted, out_dtype=out_dtype)
    check_experts(1, 1, 2, 1030, 1301, 16, unit=unit, limit=2.0, weighted=weighted, out_dtype=out_dtype)
    check_experts(2, 2, 2, 1024, 1024, 16, unit=unit, limit=2.0, weighted=weighted, out_dtype=out_dtype, sel=[-1] * 4)


def test_experts_that_the_rule_splits():
    """One token's eight experts: two CTAs a tile."""
    check_experts(1, 8, 64, 2048, 1024, 16, empty=0.0)


@pytest.mark.parametrize("D", [1001, 1100, 299, 6])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tile_rows", [16, 128])
def test_experts_whose_rows_begin_anywhere(D, out_dtype, tile_rows):
    check_experts(150, 3, 4, D, 136, tile_rows, out_dtype=out_dtype)


@pytest.mark.parametrize("D,F,unit", [(2304, 1160, "silu"), (1100, 1160, "bounded")])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_experts_of_more_tiles_than_ctas(D, F, unit, out_dtype):
    """A CTA's second tile and third: 10 column tiles of each of some 36 tiles of the plan, and 9 or 5."""
    check_experts(1100, 4, 5, D, F, 128, unit=unit, limit=2.0, out_dtype=out_dtype)


def test_few_slots_of_more_tiles_than_ctas():
    check_experts(200, 8, 64, 1152, 1160, 16)


@pytest.mark.parametrize("ranks,K", [("3", 2048), ("0", 2048), ("16", 4096), ("-2", 2048), ("many", 2048), ("", 2048), ("8", 896), ("2", 128)])
def test_ranks_that_cannot_be(monkeypatch, ranks, K):
    """A number of CTAs that the sums' exchange has no form for, or more of them than there are runs of K: refused before anything is launched."""
    from mlx_lm_b200 import ops as o

    x, w = kept(normal((4, K), 1)), kept(normal((300, K), 2))
    out, st = torch.full((4, 300), 3.0, device="cuda"), status()
    codes = o.fp8_empty(16, K, "cuda", groups=2)
    stack, plan = kept(normal((2 * 128, K), 3), 128), planned([0, 1], 2, 16, most=2)
    torch.cuda.synchronize()
    monkeypatch.setenv("MLXB_FP8_RANKS", ranks)
    with pytest.raises(o.KernelError, match="MLXB_FP8_RANKS"):
        o.linear_fp8(*x, *w, None, out, st, o.current_stream())
    with pytest.raises(o.KernelError, match="MLXB_FP8_RANKS"):
        o.moe_gemm_fp8(*codes, *stack, *plan, torch.zeros((2, 128), device="cuda"), st, o.current_stream())
    torch.cuda.synchronize()
    assert int(st) == 0 and (out == 3.0).all()
