"""Weights in 8-bit floating point: rows into codes, linear layers, the experts' products, against 64 bits."""
import math

import pytest
import torch

import fp8_refs as ref

pytestmark = pytest.mark.gpu


def ops():
    from mlx_lm_b200 import ops as o
    return o


def normal(shape, seed, dtype=torch.float32, outliers=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    if outliers and len(shape) == 2 and shape[1] > 3:
        x[:, 3::61] *= 8.0
    return x.to(dtype).cuda()


def kept(w, group_rows=None):
    o = ops()
    rows = w.shape[0] if group_rows is None else group_rows
    codes, scales = o.fp8_empty(rows, w.shape[1], w.device, groups=w.shape[0] // rows)
    o.fp8_quantize(w, codes, scales, o.current_stream(), group_rows=rows)
    return codes, scales


def status():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------ rows

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,columns,group", [(1, 1, 1), (1, 16, 1), (3, 100, 3), (5, 128, 5), (129, 513, 129), (40, 1000, 20), (300, 640, 300),
                                                (260, 1504, 130), (7, 4096, 7)])
def test_rows(rows, columns, group, dtype):
    x = normal((rows, columns), rows + columns, dtype)
    codes, scales = kept(x, group)
    want_c, want_e = ref.held(x)
    got_c, got_e = ref.read(codes, scales, columns, group)
    assert torch.equal(got_e, want_e)
    assert torch.equal(got_c, want_c)
    assert not codes.view(torch.uint8)[:, columns:].any()


def test_rows_at_the_borders():
    """Ties, the largest code, numbers just above it, subnormal codes and scales, signed zeros, and what is not finite."""
    rows = [[448.0, 1.0], [449.0, 1.0], [464.0, 29.0], [448.0 * 2 ** 100, 2.0 ** 98], [2.0 ** -140, 2.0 ** -141], [0.0, -0.0], [3.4e38, 1.0],
            [1.0, 2.0 ** -9], [256.0, 2.0 ** -10], [256.0, 1.5 * 2.0 ** -9], [256.0, 17.0], [256.0, 19.0], [-448.0, 18.0],
            [math.inf, 1.0], [-math.inf, 300.0], [math.nan, 5.0], [math.nan, math.inf]]
    x = torch.tensor(rows, dtype=torch.float32).repeat(1, 100).cuda()
    codes, scales = kept(x)
    want_c, want_e = ref.held(x)
    got_c, got_e = ref.read(codes, scales, 200, len(rows))
    assert torch.equal(got_e, want_e)
    assert torch.equal(torch.nan_to_num(got_c, nan=1e9), torch.nan_to_num(want_c, nan=1e9))


def test_rows_of_a_view():
    """Strided rows, a base that is not 16-byte aligned."""
    wide = normal((50, 700), 3, torch.bfloat16)
    for x in (wide[:, 8:8 + 512], wide[:, 1:1 + 512], wide[:, 3:3 + 130], wide[::2, 16:16 + 256]):
        codes, scales = kept(x)
        want_c, want_e = ref.held(x)
        got_c, got_e = ref.read(codes, scales, x.shape[1], x.shape[0])
        assert torch.equal(got_c, want_c) and torch.equal(got_e, want_e)


# ------------------------------------------------------------------------------------------------ linear layers

def bound(x, w, out_dtype):
    """How far a sum of K products may be off: the products are exact, each addition rounds the sum so far (and a tensor core may cut off
    what lies below 2^-24 of the largest of 32 it adds), so K 2^-23 of the sum of magnitudes bounds it; it stays far below since
    roundings cancel.  Half a step of the output's type on top."""
    K = x.shape[1]
    return (x.abs() @ w.abs().T) * (K * 2.0 ** -23 if K < 64 else 8.0 * math.sqrt(K) * 2.0 ** -23)


def check_linear(M, N, K, x_dtype=torch.bfloat16, out_dtype=torch.bfloat16, bias=False, act="none", residual=False, pad=0, seed=0):
    o = ops()
    x, w = normal((M, K), seed + 1, x_dtype), normal((N, K), seed + 2, torch.bfloat16, outliers=False) * K ** -0.5
    b = normal((N,), seed + 3) if bias else None
    room = torch.full((M, N + pad), 7.0, dtype=out_dtype, device="cuda")
    out = room[:, :N]
    res = normal((M, N), seed + 4).to(out_dtype) if residual else None
    if residual:
        out.copy_(res)
    st = status()
    xc, xs = kept(x)
    wc, ws = kept(w)
    o.linear_fp8(xc, xs, wc, ws, b, out, st, o.current_stream(), epilogue=o.ACTIVATION_CODES[act], residual=out if residual else None)
    torch.cuda.synchronize()
    assert int(st) == 0
    xv, wv = ref.values(x), ref.values(w)
    y = xv @ wv.T
    off = bound(xv, wv, out_dtype)
    if bias:
        y = y + b.double()
        off = off + y.abs() * 2.0 ** -24
    z = ref.ACTS[act](y)
    # slopes are at most 1.13 (gelu_new); its fast form is 2^-20 of its argument off at most, in bfloat16 runs
    off = 1.13 * off + (z.abs() + 1e-3) * (2.0 ** -18 if act != "none" else 0.0)
    if residual:
        z = z + res.double()
        off = off + z.abs() * 2.0 ** -24
    off = off + z.abs() * torch.finfo(out_dtype).eps / 2 + 1e-30
    err = (out.double() - z).abs()
    assert torch.isfinite(out).all()
    assert (err <= off).all(), f"{float((err / off).max())} of the bound at {M} x {N} x {K}"
    if pad:
        assert (room[:, N:] == 7.0).all()


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 32, 33, 64, 65, 127, 128])
@pytest.mark.parametrize("N,K", [(128, 128), (64, 1024), (200, 400)])
def test_linear_few_rows(M, N, K):
    check_linear(M, N, K)


@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (3, 1, 16), (16, 5, 30), (1, 129, 2100), (64, 1280, 5120), (8, 300, 8192), (1, 50257, 768), (20, 1000, 129)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_linear_few_sizes(M, N, K, out_dtype):
    check_linear(M, N, K, out_dtype=out_dtype, bias=True, residual=True)


@pytest.mark.parametrize("M,N,K", [(129, 128, 128), (256, 256, 128), (257, 300, 640), (400, 1000, 1000), (517, 1501, 1000), (1000, 136, 4096), (640, 2048, 512),
                                   (300, 40, 16), (2048, 1600, 1600)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_linear_many_sizes(M, N, K, out_dtype):
    check_linear(M, N, K, out_dtype=out_dtype)


@pytest.mark.parametrize("M,N,K", [(33, 200, 1200), (64, 300, 2048), (65, 200, 3584), (100, 1000, 4096), (128, 129, 3600), (64, 8200, 1100), (64, 8192, 1100),
                                   (48, 300, 1024), (128, 4200, 3600), (128, 4096, 3600), (100, 700, 3568)])
def test_linear_between_few_and_many(M, N, K):
    """Rows that either kernel may have, at both sides of every limit of the rule."""
    check_linear(M, N, K, bias=True)


@pytest.mark.parametrize("ranks", ["1", "2", "4", "8"])
@pytest.mark.parametrize("M", [1, 17, 40, 70])
def test_linear_few_splits(monkeypatch, ranks, M):
    """K cut among one to eight CTAs, with a last share that is shorter than the others."""
    monkeypatch.setenv("MLXB_FP8_RANKS", ranks)
    check_linear(M, 300, 2400, bias=True, act="gelu_new", residual=True)


@pytest.mark.parametrize("columns", ["128", "256"])
@pytest.mark.parametrize("pairs", ["0", "1"])
@pytest.mark.parametrize("M,N,K,pad", [(129, 300, 520, 0), (300, 1000, 128, 8), (700, 72, 2100, 3), (5000, 1400, 264, 0)])
def test_linear_many_forms(monkeypatch, columns, pairs, M, N, K, pad):
    """Every width of tile, in pairs of CTAs and not: ragged tiles, a short K, a long one, several tiles a CTA."""
    monkeypatch.setenv("MLXB_FP8_BN", columns)
    monkeypatch.setenv("MLXB_FP8_PAIR", pairs)
    check_linear(M, N, K, bias=True, pad=pad)


@pytest.mark.parametrize("M", [9, 300])
@pytest.mark.parametrize("act", ["none", "relu", "gelu_new", "tanh"])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", [False, True])
def test_linear_epilogues(M, act, out_dtype, residual):
    check_linear(M, 333, 272, out_dtype=out_dtype, bias=True, act=act, residual=residual, pad=3)


# ------------------------------------------------------------------------------------------------ experts

def planned(sel, n_experts, tile_rows, most=None):
    """A plan on the device for the choices ``sel`` (a list), with room behind it."""
    order, tiles = ref.plan(sel, n_experts, tile_rows)
    most = -(-len(sel) // tile_rows) + n_experts if most is None else most
    dev = dict(dtype=torch.int32, device="cuda")
    return (torch.tensor(order + [-1] * (len(sel) - len(order)), **dev), torch.tensor(tiles + [(-1, -1, -1)] * (most - len(tiles)), **dev),
            torch.tensor([len(tiles)], **dev), most, tile_rows)


@pytest.mark.parametrize("tile_rows", [16, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("columns", [72, 512, 1000])
def test_gather(tile_rows, dtype, columns):
    o = ops()
    T, top, E = 50, 3, 5
    g = torch.Generator().manual_seed(columns)
    sel = torch.randint(-1, E, (T * top,), generator=g).tolist()
    x = normal((T, columns), 1, dtype)
    plan = planned(sel, E, tile_rows)
    codes, scales = o.fp8_empty(tile_rows, columns, "cuda", groups=plan[3])
    codes.view(torch.uint8).fill_(1)
    scales.fill_(2)
    o.moe_gather_fp8(x, top, *plan, codes, scales, o.current_stream())
    got_c, got_e = ref.read(codes, scales, columns, tile_rows)
    order, tiles = ref.plan(sel, E, tile_rows)
    touched = torch.zeros(codes.shape[0], dtype=torch.bool, device="cuda")
    for t, (_, first, n) in enumerate(tiles):
        rows = torch.tensor([s // top for s in order[first:first + n]], device="cuda")
        want_c, want_e = ref.held(x[rows])
        assert torch.equal(got_c[t * tile_rows:t * tile_rows + n], want_c)
        assert torch.equal(got_e[t * tile_rows:t * tile_rows + n], want_e)
        touched[t * tile_rows:t * tile_rows + n] = True
    assert (codes.view(torch.uint8)[~touched] == 1).all()


def check_experts(T, top, E, D, F, tile_rows, unit="silu", limit=0.0, weighted=True, out_dtype=torch.float32, seed=0, sel=None, empty=0.1):
    """Both products; the hidden rows are taken from the device for the second, so that each is held to its own bound."""
    o = ops()
    g = torch.Generator().manual_seed(seed)
    if sel is None:
        sel = [-1 if torch.rand((), generator=g) < empty else int(torch.randint(0, E, (), generator=g)) for _ in range(T * top)]
    S = T * top
    x = normal((T, D), seed + 1, torch.bfloat16)
    w_in = normal((E * 2 * F, D), seed + 2, torch.bfloat16, outliers=False) * D ** -0.5
    w_out = normal((E * D, F), seed + 3, torch.bfloat16, outliers=False) * F ** -0.5
    weight = torch.rand(S, generator=g).cuda() if weighted else None
    plan = planned(sel, E, tile_rows)
    order, tiles = ref.plan(sel, E, tile_rows)
    codes, scales = o.fp8_empty(tile_rows, D, "cuda", groups=plan[3])
    hc, hs = o.fp8_empty(tile_rows, F, "cuda", groups=plan[3])
    st, out = status(), torch.full((S, D), 3.0, dtype=out_dtype, device="cuda")
    stream = o.current_stream()
    wi, wo = kept(w_in, F), kept(w_out, D)
    o.moe_gather_fp8(x, top, *plan, codes, scales, stream)
    o.moe_gemm_fp8(codes, scales, *wi, *plan, hc, st, stream, sel_weight=weight, gated=True, out_scales=hs, unit=unit, limit=limit)
    o.moe_gemm_fp8(hc, hs, *wo, *plan, out, st, stream)
    torch.cuda.synchronize()
    assert int(st) == 0
    xv, wiv, wov = ref.values(x), ref.values(w_in).view(E, 2, F, D), ref.values(w_out).view(E, D, F)
    h_all, (_, h_exp) = ref.numbers(hc, hs, F, tile_rows), ref.read(hc, hs, F, tile_rows)
    written = torch.zeros(S, dtype=torch.bool, device="cuda")
    for t, (e, first, n) in enumerate(tiles):
        slots = torch.tensor(order[first:first + n], device="cuda")
        rows = xv[slots // top]
        gate, up = rows @ wiv[e, 0].T, rows @ wiv[e, 1].T
        wgt = (weight[slots] if weighted else torch.ones(n, device="cuda")).double()[:, None]
        h = ref.unit(unit, gate, up, wgt, limit)
        got_h = h_all[t * tile_rows:t * tile_rows + n]
        # the float32 sums' bound through the unit (its slopes are below 1.1 |w| (1 + |the other factor|)), then half a step of the code: 2^-4
        # of the value, or 2^-10 of the scale below 2^-6 of it; a scale one power up where a float32 magnitude crossed its border
        off = 1.2 * wgt * (bound(rows, wiv[e, 0], None) * (1 + up.abs()) + bound(rows, wiv[e, 1], None) * (1 + gate.abs())) + h.abs() * 2.0 ** -20
        scale = torch.ldexp(torch.ones_like(h), h_exp[t * tile_rows:t * tile_rows + n].repeat_interleave(ref.RUN, 1)[:, :F])
        err = (got_h - h).abs()
        assert (err <= off + torch.maximum((h.abs() + off) * 2.0 ** -4, scale * 2.0 ** -10)).all(), (t, float(err.max()))
        top_h = torch.nn.functional.pad(h.abs(), (0, -F % ref.RUN)).view(n, -1, ref.RUN).amax(-1)
        got_scale = torch.ldexp(torch.ones_like(top_h), h_exp[t * tile_rows:t * tile_rows + n])
        assert (top_h <= 448.0 * got_scale * (1 + 1e-4)).all() and ((top_h >= 224.0 * got_scale * (1 - 1e-4)) | (top_h == 0)).all()
        y = got_h @ wov[e].T
        got = out[slots].double()
        assert ((got - y).abs() <= bound(got_h, wov[e], None) + y.abs() * torch.finfo(out_dtype).eps / 2 + 1e-30).all(), t
        written[slots] = True
    assert (out[~written] == 3.0).all()


@pytest.mark.parametrize("tile_rows", [16, 128])
@pytest.mark.parametrize("D,F", [(128, 128), (256, 640), (200, 72), (1000, 520), (2048, 768)])
def test_experts(tile_rows, D, F):
    check_experts(37, 3, 6, D, F, tile_rows)


@pytest.mark.parametrize("T,top,E,tile_rows", [(1, 1, 1, 16), (1, 8, 64, 16), (2, 2, 2, 128), (64, 8, 8, 128), (300, 4, 16, 128),
                                               (500, 2, 3, 16), (700, 1, 2, 16), (90, 8, 40, 128)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_experts_counts(T, top, E, tile_rows, out_dtype):
    check_experts(T, top, E, 384, 272, tile_rows, out_dtype=out_dtype, seed=T)


@pytest.mark.parametrize("tile_rows", [16, 128])
@pytest.mark.parametrize("unit,weighted", [("silu", False), ("bounded", True), ("bounded", False)])
def test_experts_units(tile_rows, unit, weighted):
    check_experts(40, 2, 4, 256, 200, tile_rows, unit=unit, limit=2.0, weighted=weighted)


@pytest.mark.parametrize("tile_rows", [16, 128])
def test_experts_of_one_and_of_nobody(tile_rows):
    """All slots on one expert; all but one slot on nobody; none at all."""
    check_experts(60, 2, 5, 256, 128, tile_rows, sel=[3] * 120)
    check_experts(60, 2, 5, 256, 128, tile_rows, sel=[-1] * 119 + [4])
    check_experts(60, 2, 5, 256, 128, tile_rows, sel=[-1] * 120)


# ------------------------------------------------------------------------------------------------ how they are used

@pytest.mark.parametrize("act", ["none", "relu", "gelu_new", "tanh"])
def test_a_row_that_is_not_finite_keeps_to_itself(act):
    o = ops()
    for M in (20, 300):
        x = normal((M, 400), 1, torch.bfloat16)
        x[3, 17], x[5, 399], x[9, 0] = math.nan, math.inf, -math.inf
        w = normal((260, 400), 2, torch.bfloat16) * 0.05
        out, st = torch.zeros((M, 260), dtype=torch.bfloat16, device="cuda"), status()
        o.linear_fp8(*kept(x), *kept(w), None, out, st, o.current_stream(), epilogue=o.ACTIVATION_CODES[act])
        bad = torch.isnan(out).all(1)
        assert bad.nonzero().view(-1).tolist() == [3, 5, 9] and torch.isfinite(out[~bad]).all()


@pytest.mark.parametrize("tile_rows", [16, 128])
@pytest.mark.parametrize("unit", ["silu", "bounded"])
def test_a_slot_that_is_not_finite_keeps_to_itself(tile_rows, unit):
    o = ops()
    T, E, D, F = 30, 2, 256, 200
    x = normal((T, D), 1, torch.bfloat16)
    x[4, 100], x[7] = math.inf, math.nan
    wi, wo = kept(normal((E * 2 * F, D), 2, torch.bfloat16) * 0.06, F), kept(normal((E * D, F), 3, torch.bfloat16) * 0.06, D)
    plan = planned([i % 2 for i in range(T)], E, tile_rows)
    codes, scales = o.fp8_empty(tile_rows, D, "cuda", groups=plan[3])
    hc, hs = o.fp8_empty(tile_rows, F, "cuda", groups=plan[3])
    out, st, stream = torch.zeros((T, D), device="cuda"), status(), o.current_stream()
    o.moe_gather_fp8(x, 1, *plan, codes, scales, stream)
    o.moe_gemm_fp8(codes, scales, *wi, *plan, hc, st, stream, gated=True, out_scales=hs, unit=unit, limit=2.0)
    o.moe_gemm_fp8(hc, hs, *wo, *plan, out, st, stream)
    bad = torch.isnan(out).any(1)
    assert bad.nonzero().view(-1).tolist() == [4, 7]


def test_weights_quantised_right_before_they_are_read():
    """The product right behind fp8_quantize of its own weights, again and again on other ones: never the ones before."""
    o = ops()
    for N in (100, 128, 129, 1000):
        x = normal((4, 2048), 1, torch.bfloat16)
        w = [normal((N, 2048), 2 + i, torch.bfloat16) for i in range(4)]
        want = [ref.values(x) @ ref.values(m).T for m in w]
        xc, (wc, ws) = kept(x), o.fp8_empty(N, 2048, "cuda")
        outs, st = [torch.zeros((4, N), device="cuda") for _ in w], status()
        torch.cuda.synchronize()
        for m, out in zip(w * 5, outs * 5):
            o.fp8_quantize(m, wc, ws, o.current_stream())
            o.linear_fp8(*xc, wc, ws, None, out, st, o.current_stream())
        for out, y in zip(outs, want):
            assert float((out.double() - y).abs().max()) <= 1e-3 * float(y.abs().max())


@pytest.mark.parametrize("M", [4, 200])
def test_weights_quantised_in_blocks_right_before_they_are_read(M):
    """A weight that is rounded 128 rows a call, first to last and last to first, and read by the launch behind the last of them."""
    o = ops()
    N, K = 1024, 2048
    x = normal((M, K), 1, torch.bfloat16)
    xc, (wc, ws) = kept(x), o.fp8_empty(N, K, "cuda")
    w = [normal((N, K), 2 + i, torch.bfloat16) for i in range(6)]
    outs, st = [torch.zeros((M, N), device="cuda") for _ in w], status()

    def step():
        for turn, (m, out) in enumerate(zip(w, outs)):
            for b in range(0, N, 128) if turn & 1 else range(N - 128, -1, -128):
                o.fp8_quantize(m[b:b + 128], wc[b:b + 128], ws[:, b // 128:b // 128 + 1], o.current_stream())
            o.linear_fp8(*xc, wc, ws, None, out, st, o.current_stream())

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    for out in outs:
        out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for m, out in zip(w, outs):
        y = ref.values(x) @ ref.values(m).T
        assert float((out.double() - y).abs().max()) <= 1e-4 * float(y.abs().max())
    assert int(st) == 0


@pytest.mark.parametrize("M", [5, 300])
def test_captured_and_replayed(M):
    """A graph of both calls, replayed on other rows; beside it another graph with rows of its own."""
    o = ops()
    w, st = kept(normal((500, 640), 9, torch.bfloat16) * 0.04), status()
    wv = ref.values(normal((500, 640), 9, torch.bfloat16) * 0.04)
    sets = []
    for i in range(2):
        x, out = normal((M, 640), i, torch.bfloat16), torch.zeros((M, 500), device="cuda")
        codes, scales = o.fp8_empty(M, 640, "cuda")
        def step(x=x, out=out, codes=codes, scales=scales):
            o.fp8_quantize(x, codes, scales, o.current_stream())
            o.linear_fp8(codes, scales, *w, None, out, st, o.current_stream())
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        sets.append((x, out, graph))
    for turn in range(3):
        for i, (x, out, graph) in enumerate(sets):
            x.copy_(normal((M, 640), 50 + 2 * turn + i, torch.bfloat16))
        streams = [torch.cuda.Stream() for _ in sets]
        torch.cuda.synchronize()
        for s, (_, _, graph) in zip(streams, sets):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for x, out, _ in sets:
            y = ref.values(x) @ wv.T
            assert float((out.double() - y).abs().max()) <= 1e-4 * float(y.abs().max())
    assert int(st) == 0


def test_the_whole_feed_forward_captured():
    """Router, gather and both products in one graph, replayed on other tokens: the choices, and rows of a plain computation."""
    o = ops()
    T, E, top, D, F = 40, 16, 3, 256, 200
    S = T * top
    w_in, w_out = normal((E * 2 * F, D), 1, torch.bfloat16) * D ** -0.5, normal((E * D, F), 2, torch.bfloat16) * F ** -0.5
    wi, wo = kept(w_in, F), kept(w_out, D)
    rows = o.moe_fp8_tile_rows(S, E)
    most = o.moe_max_tiles(S, E, rows)
    i = dict(dtype=torch.int32, device="cuda")
    x, logits = torch.zeros((T, D), dtype=torch.bfloat16, device="cuda"), torch.zeros((T, E), device="cuda")
    sel, weight, order, tiles, n = torch.zeros(S, **i), torch.zeros(S, device="cuda"), torch.zeros(S, **i), torch.zeros((most, 3), **i), torch.zeros(1, **i)
    scratch, st, out = torch.zeros(o.moe_route_scratch(T, E), **i), status(), torch.zeros((S, D), device="cuda")
    (c, s), (hc, hs) = o.fp8_empty(rows, D, "cuda", groups=most), o.fp8_empty(rows, F, "cuda", groups=most)

    def step():
        stream, plan = o.current_stream(), (order, tiles, n, most, rows)
        o.moe_route_plan(logits, None, top, sel, weight, rows, order, tiles, n, scratch, stream, score="softmax", renormalize=True)
        o.moe_gather_fp8(x, top, *plan, c, s, stream)
        o.moe_gemm_fp8(c, s, *wi, *plan, hc, st, stream, sel_weight=weight, gated=True, out_scales=hs)
        o.moe_gemm_fp8(hc, hs, *wo, *plan, out, st, stream)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    wiv, wov = ref.values(w_in).view(E, 2, F, D), ref.values(w_out).view(E, D, F)
    for turn in range(3):
        x.copy_(normal((T, D), 10 + turn, torch.bfloat16))
        logits.copy_(normal((T, E), 20 + turn))
        graph.replay()
        torch.cuda.synchronize()
        want, w = ref.route(logits.cpu(), [True] * T, top, score="softmax", renormalize=True)
        assert sel.tolist() == [e for row in want for e in row]
        xv = ref.values(x)
        for t in range(T):
            for k, e in enumerate(want[t]):
                h = ref.values(ref.unit("silu", xv[t:t + 1] @ wiv[e, 0].T, xv[t:t + 1] @ wiv[e, 1].T, w[t][k], 0.0).float())
                y = (h @ wov[e].T)[0]
                # a hidden number that falls on the other side of a border of codes is 2^-3 of itself off, one of 200
                assert float((out[t * top + k].double() - y).norm() / y.norm()) <= 1e-2
    assert int(st) == 0


def test_nothing_to_do():
    o = ops()
    st, stream = status(), o.current_stream()
    i = dict(dtype=torch.int32, device="cuda")
    w = kept(normal((64, 128), 1, torch.bfloat16))
    empty = torch.zeros((0, 128), dtype=torch.bfloat16, device="cuda")
    some = o.fp8_empty(16, 128, "cuda", groups=4)
    o.fp8_quantize(empty, *some, stream)
    o.linear_fp8(*some, *w, None, torch.zeros((0, 64), device="cuda"), st, stream)
    none, tiles, n = torch.zeros(0, **i), torch.full((4, 3), -1, **i), torch.full((1,), 9, **i)
    o.moe_route_plan(torch.zeros((0, 4), device="cuda"), None, 2, none, torch.zeros(0, device="cuda"), 16, none, tiles, n, torch.zeros(1, **i), stream)
    assert int(n) == 0 and (tiles == -1).all()
    o.moe_gather_fp8(empty, 2, none, tiles, n, 4, 16, *some, stream)
    o.moe_gemm_fp8(*some, *kept(normal((4 * 32, 128), 1, torch.bfloat16), 32), none, tiles, n, 4, 16, torch.zeros((0, 32), device="cuda"), st, stream)
    torch.cuda.synchronize()
    assert int(st) == 0


def test_a_plan_with_numbers_out_of_range_reaches_nothing():
    """Places, slots and experts that do not exist, and a tile longer than tiles are: left out or held to what there is, on the host's word for sizes."""
    o = ops()
    E, D, F, S = 3, 128, 96, 20
    i = dict(dtype=torch.int32, device="cuda")
    x = normal((S, D), 1, torch.bfloat16)
    wi, wo = kept(normal((E * 2 * F, D), 2, torch.bfloat16), F), kept(normal((E * D, F), 3, torch.bfloat16), D)
    for rows in (16, 128):
        most = 5
        order = torch.tensor([0, 1, -5, 10 ** 9] + list(range(4, S)), **i)
        tiles = torch.tensor([[0, 0, 4], [99, 4, 3], [-7, 7, 3], [1, 15, 2000], [2, 10 ** 9, 4]], **i)
        n = torch.tensor([5], **i)
        (c, s), (hc, hs) = o.fp8_empty(rows, D, "cuda", groups=most), o.fp8_empty(rows, F, "cuda", groups=most)
        out, st, stream = torch.full((S, D), 5.0, device="cuda"), status(), o.current_stream()
        plan = (order, tiles, n, most, rows)
        o.moe_gather_fp8(x, 1, *plan, c, s, stream)
        o.moe_gemm_fp8(c, s, *wi, *plan, hc, st, stream, sel_weight=torch.ones(S, device="cuda"), gated=True, out_scales=hs)
        o.moe_gemm_fp8(hc, hs, *wo, *plan, out, st, stream)
        torch.cuda.synchronize()
        assert (out[2:4] == 5.0).all() and not (out[:2] == 5.0).all(1).any()
        assert torch.isfinite(out).all() and int(st) == 0


def test_codes_beyond_2_31_bytes():
    """More codes than 32 bits count, the last rows among those that are looked at."""
    o = ops()
    N, K = 70000, 32768
    codes, scales = o.fp8_empty(N, K, "cuda")
    w = torch.empty((N, K), dtype=torch.bfloat16, device="cuda")
    for a in range(0, N, 10000):
        w[a:a + 10000].normal_(generator=torch.Generator(device="cuda").manual_seed(a))
    o.fp8_quantize(w, codes, scales, o.current_stream())
    at = torch.tensor([0, 1, 65535, 65536, 65537, N - 129, N - 1], device="cuda")
    few = ref.values(w[at])
    del w
    for M in (3, 200):
        x = normal((M, K), 1, torch.bfloat16)
        out, st = torch.zeros((M, N), device="cuda"), status()
        o.linear_fp8(*kept(x), codes, scales, None, out, st, o.current_stream())
        y = ref.values(x) @ few.T
        assert float((out[:, at].double() - y).abs().max()) <= 1e-4 * float(y.abs().max())
        assert int(st) == 0


@pytest.mark.parametrize("name,M,N,K", [("fp8_few", 5, 40000, 512), ("fp8_few", 5, 512, 2048), ("fp8_many", 300, 300, 512), ("fp8_many", 100, 300, 512)])
def test_a_wait_that_runs_out(name, M, N, K):
    """An arrival that never comes (left out by the test's build): the kernel comes back by itself, says so and has written nothing; the next launch is right."""
    from ctypes import c_int

    from mlx_lm_b200.ops import build

    o = ops()
    lib_name = name + ":MLXB_TEST_WAIT_TIMEOUT=1"
    lib = build.load(lib_name)
    lib.mlxb_test_withhold_arrival.argtypes, lib.mlxb_test_withhold_arrival.restype = [c_int], c_int
    x, w = normal((M, K), 1, torch.bfloat16), normal((N, K), 2, torch.bfloat16) * 0.05
    (xc, xs), (wc, ws) = kept(x), kept(w)
    out, st = torch.zeros((M, N), device="cuda"), status()

    def launch():
        o._call(lib_name, "mlxb_fp8_linear_few" if name == "fp8_few" else "mlxb_fp8_linear_many", o._FP8_ARGS, *o._fp8_linear_record(
            xc.data_ptr(), xs.data_ptr(), wc.data_ptr(), ws.data_ptr(), 0, 0, out.data_ptr(), st.data_ptr(), True, M, N, K, N, 0), o.current_stream())
        torch.cuda.synchronize()

    assert lib.mlxb_test_withhold_arrival(1) == 0
    try:
        launch()
        assert int(st) == o.ST_WAIT_TIMEOUT
        if N < 40000:                      # more tiles than CTAs: only each one's first is lost
            assert not out.any()
    finally:
        assert lib.mlxb_test_withhold_arrival(0) == 0
    st.zero_()
    launch()
    y = ref.values(x) @ ref.values(w).T
    assert int(st) == 0 and float((out.double() - y).abs().max()) <= 1e-4 * float(y.abs().max())
