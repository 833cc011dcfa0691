"""What the operators for weights in 8-bit floating point and the router with its plan refuse, on the CPU: nothing gets as far as a launch."""
import pytest
import torch

from mlx_lm_b200 import ops
from mlx_lm_b200.ops import KernelError


def pair(rows=20, columns=200, groups=1):
    return ops.fp8_empty(rows, columns, "cpu", groups=groups)


def test_memory_of_a_matrix():
    codes, scales = ops.fp8_empty(130, 1000, "cpu", groups=3)
    assert codes.shape == (390, 1008) and codes.dtype == torch.float8_e4m3fn
    assert scales.shape == (3, 2, 2, 512) and scales.dtype == torch.uint8
    for bad in ((0, 5), (5, 0), (5, 5, 0)):
        with pytest.raises(KernelError):
            ops.fp8_empty(bad[0], bad[1], "cpu", *bad[2:])


@pytest.mark.parametrize("x,target,kw", [
    (torch.zeros(20, 200, dtype=torch.float16), pair(), {}),
    (torch.zeros(20), pair(), {}),
    (torch.zeros(200, 20).t(), pair(), {}),
    (torch.zeros(1, 200).expand(20, 200), pair(), {}),
    (torch.zeros(21, 200), pair(), {}),
    (torch.zeros(20, 210), pair(), {}),
    (torch.zeros(20, 200), pair(20, 700), {}),
    (torch.zeros(20, 200), pair(), dict(group_rows=7)),
    (torch.zeros(20, 200), pair(10, 200, 2), {}),
    (torch.zeros(20, 200), (pair()[0].view(torch.uint8), pair()[1]), {}),
    (torch.zeros(20, 200), (pair()[0], pair()[1][:, :, :, :256]), {}),
    (torch.zeros(20, 200), (pair(20, 400)[0][:, :208], pair()[1]), {}),
    (torch.zeros(20, 200), pair(), {}),                       # all right, but on the CPU
])
def test_quantize(x, target, kw):
    with pytest.raises(KernelError, match="fp8_quantize"):
        ops.fp8_quantize(x, *target, 0, **kw)


def linear(M=20, N=30, K=200, **change):
    a = dict(x=pair(M, K), w=pair(N, K), bias=torch.zeros(N), out=torch.zeros(M, N), status=torch.zeros(1, dtype=torch.int32), residual=None)
    a.update(change)
    ops.linear_fp8(*a["x"], *a["w"], a["bias"], a["out"], a["status"], 0, residual=a["residual"])


@pytest.mark.parametrize("change", [
    dict(x=pair(21, 200)), dict(x=pair(20, 216)), dict(w=pair(31, 200)), dict(w=pair(15, 200, 2)), dict(bias=torch.zeros(29)),
    dict(bias=torch.zeros(30, dtype=torch.bfloat16)), dict(bias=torch.zeros(60)[::2]), dict(out=torch.zeros(20, 30, dtype=torch.float16)),
    dict(out=torch.zeros(30, 20).t()), dict(status=torch.zeros(1)), dict(residual=torch.zeros(20, 30, dtype=torch.bfloat16)),
    dict(residual=torch.zeros(20, 31)), dict(residual=torch.zeros(20, 40)[:, :30]), {}])
def test_linear(change):
    with pytest.raises(KernelError, match="8 bits"):
        linear(**change)


def plan(S=40, E=4, rows=16, **change):
    most = ops.moe_max_tiles(S, E, rows)
    p = dict(order=torch.zeros(S, dtype=torch.int32), tiles=torch.zeros(most, 3, dtype=torch.int32), n=torch.zeros(1, dtype=torch.int32), most=most, rows=rows)
    p.update(change)
    return tuple(p.values())


@pytest.mark.parametrize("x,a_div,p,target", [
    (torch.zeros(20, 200), 2, plan(rows=24), pair(24, 200, 10)),
    (torch.zeros(20, 200), 2, plan(), pair(16, 200, 5)),
    (torch.zeros(20, 200), 2, plan(), pair(16, 300, 10)),
    (torch.zeros(19, 200), 2, plan(), pair(16, 200, 10)),
    (torch.zeros(20, 200), 0, plan(), pair(16, 200, 10)),
    (torch.zeros(20, 200), 2, plan(order=torch.zeros(40)), pair(16, 200, 10)),
    (torch.zeros(20, 200), 2, plan(tiles=torch.zeros(2, 3, dtype=torch.int32)), pair(16, 200, 10)),
    (torch.zeros(20, 200), 2, plan(n=torch.zeros(0, dtype=torch.int32)), pair(16, 200, 10)),
    (torch.zeros(20, 200), 2, plan(), pair(16, 200, 10)),
])
def test_gather(x, a_div, p, target):
    with pytest.raises(KernelError, match="moe_gather_fp8"):
        ops.moe_gather_fp8(x, a_div, *p, *target, 0)


def experts(gated=True, p=None, **change):
    p = plan() if p is None else p
    a = dict(x=pair(16, 200, 10), w=pair(96, 200, 8 if gated else 4), out=pair(16, 96, 10) if gated else (torch.zeros(40, 96), None),
             weight=torch.zeros(40) if gated else None, status=torch.zeros(1, dtype=torch.int32), unit="silu")
    a.update(change)
    ops.moe_gemm_fp8(*a["x"], *a["w"], *p, a["out"][0], a["status"], 0, sel_weight=a["weight"], gated=gated, out_scales=a["out"][1], unit=a["unit"])


@pytest.mark.parametrize("gated,change", [
    (True, dict(w=pair(96, 200, 7))), (True, dict(w=pair(96, 300, 8))), (True, dict(x=pair(16, 200, 9))), (True, dict(x=pair(32, 200, 10))),
    (True, dict(out=pair(16, 96, 9))), (True, dict(out=pair(16, 200, 10))), (True, dict(out=(pair(16, 96, 10)[0], None))),
    (True, dict(weight=torch.zeros(39))), (True, dict(weight=torch.zeros(40, dtype=torch.float64))), (True, dict(unit="relu")),
    (True, dict(status=torch.zeros(1))), (True, {}), (False, dict(out=(torch.zeros(39, 96), None))), (False, dict(out=(torch.zeros(40, 95), None))),
    (False, dict(out=(torch.zeros(40, 96, dtype=torch.float16), None))), (False, dict(p=plan(rows=256))), (False, {})])
def test_experts(gated, change):
    with pytest.raises(KernelError, match="moe_gemm_fp8"):
        experts(gated, **change)


def route(T=10, E=32, top=4, rows=16, **change):
    S, i = T * top, dict(dtype=torch.int32)
    a = dict(logits=torch.zeros(T, E), req=None, sel=torch.zeros(S, **i), weight=torch.zeros(S), order=torch.zeros(S, **i),
             tiles=torch.zeros(S + E, 3, **i), n=torch.zeros(1, **i), scratch=torch.zeros(4096, **i))
    options = {k: v for k, v in change.items() if k not in a}
    a.update({k: v for k, v in change.items() if k in a})
    ops.moe_route_plan(a["logits"], a["req"], top, a["sel"], a["weight"], rows, a["order"], a["tiles"], a["n"], a["scratch"], 0, **options)


@pytest.mark.parametrize("change", [
    dict(top=0), dict(top=33), dict(E=1025), dict(E=2000, top=65), dict(groups=5), dict(groups=8, keep_groups=9), dict(groups=8, keep_groups=0),
    dict(groups=8, keep_groups=1, top=5), dict(E=512, groups=256, keep_groups=2), dict(identity=32), dict(identity=-1), dict(rows=0), dict(score="tanh"),
    dict(group_score="three"), dict(logits=torch.zeros(10, 32, dtype=torch.bfloat16)), dict(logits=torch.zeros(32, 10).t()),
    dict(req=torch.zeros(9, dtype=torch.int32)), dict(sel=torch.zeros(39, dtype=torch.int32)), dict(weight=torch.zeros(40, dtype=torch.int32)),
    dict(order=torch.zeros(80, dtype=torch.int32)[::2]), dict(tiles=torch.zeros(30, 3, dtype=torch.int32)), dict(n=torch.zeros(1)),
    dict(correction=torch.zeros(31)), {}])
def test_route(change):
    with pytest.raises(KernelError, match="moe_route_plan"):
        route(**change)


def test_tile_rows_follow_the_slots_of_an_expert():
    assert [ops.moe_fp8_tile_rows(n, 16) for n in (1, 128, 129, 256, 100000)] == [16, 16, 128, 128, 128]


def test_parts():
    from mlx_lm_b200.parts.feed_forward import ExpertsMLP
    from mlx_lm_b200.parts.linear import Linear

    with pytest.raises(ValueError, match="judged"):
        ExpertsMLP("ff", 64, 32, 8, 2, groups=(2, 1), group_score="all")
    with pytest.raises(ValueError, match="judged"):
        ExpertsMLP("ff", 64, 32, 2048, 2, groups=(2, 1), group_score="two")
    part = ExpertsMLP("ff", 256, 128, 8, 2)
    assert "moe_router" not in part.kernel_libs
    part.set_weight_bits(8)
    assert "moe_router" in part.kernel_libs and part.router.weight_bits == 8 and not part.router.in_eight_bits()
    for n_in, n_out, held in ((128, 128, True), (127, 500, False), (500, 127, False)):
        linear = Linear("l", n_in, n_out)
        assert not linear.in_eight_bits()
        linear.set_weight_bits(8)
        assert linear.in_eight_bits() is held


def test_command_lines():
    import importlib

    benchmark, generate = (importlib.import_module("mlx_lm_b200." + name) for name in ("benchmark", "generate"))
    assert generate.setup_arg_parser().parse_args([]).weight_bits is None
    assert generate.setup_arg_parser().parse_args(["--weight-bits", "8"]).weight_bits == 8
    assert benchmark.setup_arg_parser().parse_args(["--model", "m", "--weight-bits", "8"]).weight_bits == 8
    with pytest.raises(SystemExit):
        generate.setup_arg_parser().parse_args(["--weight-bits", "4"])
