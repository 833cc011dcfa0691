"""Operators for weights in 8-bit floating point, as cases that can be timed and compared.

A row of ``K`` numbers is held as e4m3 codes with one scale ``2**e`` for each run of 128 columns; ``e`` is the least whole number with
``largest finite magnitude <= 448 * 2**e`` (within -127 .. 127), a code is ``x * 2**-e`` rounded to nearest, ties to even.

``linear``    ``act(x W^T + bias) (+ residual)``: W was laid out that way once, the rows of x are within the call.  Sums are float32.
``experts``   a feed-forward of many small gated experts: the router chooses (as in ``route``), every (token, choice) slot goes through
              ``h = silu(w g) * (w u)`` with ``g`` and ``u`` the products of the token's row with the expert's gate and up rows and ``w`` the
              slot's weight, then ``h``, held in 8 bits like any row, through the expert's down rows.  Outputs: the choices, their weights and
              a row for every slot.
``route``     scores ``sigmoid(z)`` or ``softmax(z)``; a correction for each expert goes on for the choice only; neighbouring experts form
              groups, judged by the sum of their two best choice scores, of which the best few stay; the ``top`` best are chosen (ties: the lower
              index), their scores divided by their sum are the weights.  Then the plan of the experts' products: slots sorted by expert
              and, within one, by number, and tiles of at most ``tile`` slots of one expert (expert, first place, slots).

Sizes: widths of the configurations of this repository (1024 to 1600 and four times that) and generic ones up to 8192; 8 to 256
experts of which 1 to 8 are chosen; 1 to 8192 tokens a step.
"""
import math

import torch

own = False

BLOCK = 128
SCALE = 2.5           # what the router multiplies every weight by


# ------------------------------------------------------------------------------------------------ the cases

def listed():
    return [
        # one user's chat: a token at a time through a square projection
        dict(name="linear 1 of 4096x4096", kind="linear", rows=1, inner=4096, outer=4096, x="bfloat16", out="bfloat16", bias=False, act="none",
             residual=False),
        # a few users: the wide projection of a feed-forward
        dict(name="linear 8 of 4096x14336", kind="linear", rows=8, inner=4096, outer=14336, x="bfloat16", out="bfloat16", bias=False, act="none",
             residual=False),
        # a full decode batch: the second projection of GPT-2 large's feed-forward, added to a float32 stream
        dict(name="linear 64 of 5120x1280", kind="linear", rows=64, inner=5120, outer=1280, x="bfloat16", out="float32", bias=True, act="none",
             residual=True),
        # a short prompt through a layer of odd sizes
        dict(name="linear 517 of 1000x1501", kind="linear", rows=517, inner=1000, outer=1501, x="bfloat16", out="bfloat16", bias=True,
             act="relu", residual=False),
        # a prompt through the first projection of GPT-2 XL's feed-forward
        dict(name="linear 2048 of 1600x6400", kind="linear", rows=2048, inner=1600, outer=6400, x="bfloat16", out="bfloat16", bias=True,
             act="gelu_new", residual=False),
        # many prompts at once through a large model's square projection
        dict(name="linear 8192 of 8192x8192", kind="linear", rows=8192, inner=8192, outer=8192, x="bfloat16", out="bfloat16", bias=False,
             act="none", residual=True),
        # one user's chat with a mixture of experts
        dict(name="experts 1 token 8 of 64", kind="experts", tokens=1, experts=64, top=8, width=2048, inner=1024, score="softmax", groups=1,
             keep=1, correction=False, live=1.0),
        # a decode batch, most experts are met
        dict(name="experts 32 tokens 8 of 128", kind="experts", tokens=32, experts=128, top=8, width=2048, inner=768, score="sigmoid",
             groups=8, keep=4, correction=True, live=1.0),
        # a short prompt, odd sizes, rows that pad the step
        dict(name="experts 300 tokens 4 of 16", kind="experts", tokens=300, experts=16, top=4, width=1000, inner=520, score="sigmoid",
             groups=1, keep=1, correction=True, live=0.9),
        # prompts
        dict(name="experts 4096 tokens 8 of 64", kind="experts", tokens=4096, experts=64, top=8, width=2048, inner=1024, score="softmax",
             groups=1, keep=1, correction=False, live=1.0),
        # a decode batch's choice of experts
        dict(name="route 64 of 256", kind="route", tokens=64, experts=256, top=8, score="sigmoid", groups=8, keep=4, correction=True, tile=16,
             live=1.0),
        # a prompt's
        dict(name="route 8192 of 256", kind="route", tokens=8192, experts=256, top=8, score="sigmoid", groups=8, keep=4, correction=True,
             tile=128, live=1.0),
    ]


MOST_LINEAR = 8192 ** 3
MOST_EXPERTS = 4096 * 8 * 2048 * 1024


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _router(rng, case):
    E = case["experts"] = rng.choice([8, 16, 24, 60, 64, 96, 128, 160, 256])
    case["score"] = rng.choice(["sigmoid", "softmax"])
    case["groups"] = rng.choice([g for g in (1, 1, 4, 8) if E // g >= 2 and E % g == 0])
    case["keep"] = max(1, case["groups"] // 2)
    case["top"] = rng.randint(1, min(8, E // case["groups"] * case["keep"]))
    case["correction"] = case["groups"] > 1 or rng.random() < 0.5
    case["live"] = 1.0 if rng.random() < 0.7 else 0.9


def draw(rng):
    kind = rng.choice(["linear", "linear", "experts", "route"])
    case = dict(kind=kind)
    if kind == "linear":
        case["inner"], case["outer"] = (rng.choice([8, 8, 16, 1]) * _spread(rng, 16, 1024) for _ in range(2))
        case["rows"] = _spread(rng, 1, max(1, min(8192, MOST_LINEAR // (case["inner"] * case["outer"]))))
        case["x"] = "float32" if rng.random() < 0.15 else "bfloat16"
        case["out"] = rng.choice(["bfloat16", "bfloat16", "float32"])
        case["bias"], case["residual"] = rng.random() < 0.5, rng.random() < 0.3
        case["act"] = rng.choice(["none", "none", "gelu_new", "relu"])
    elif kind == "experts":
        _router(rng, case)
        case["width"], case["inner"] = 8 * _spread(rng, 16, 512), 8 * _spread(rng, 8, 256)
        while case["experts"] * case["width"] * case["inner"] > 64 * 2048 * 2048:
            case["inner"] = max(64, case["inner"] // 16 * 8)
            case["width"] = max(128, case["width"] // 16 * 8)
        case["tokens"] = _spread(rng, 1, max(1, min(4096, MOST_EXPERTS // (case["top"] * case["width"] * case["inner"]))))
    else:
        _router(rng, case)
        case["tokens"] = _spread(rng, 1, 8192)
        case["tile"] = rng.choice([16, 32, 64, 128])
    return case


# ------------------------------------------------------------------------------------------------ inputs

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case=case, status=torch.zeros(1, dtype=torch.int32, device=dev))

    def rows(n, width, dtype):
        # what a norm leaves: normal numbers, some columns much larger than others
        size = torch.ones(width, device=dev)
        size[3::61] = 8.0
        return (torch.randn((n, width), generator=g, device=dev) * size).to(dtype)

    def weights(*shape):
        return (torch.randn(shape, generator=g, device=dev) * shape[-1] ** -0.5).to(torch.bfloat16)

    if case["kind"] == "linear":
        M, K, N = case["rows"], case["inner"], case["outer"]
        out = getattr(torch, case["out"])
        s["x"] = rows(M, K, getattr(torch, case["x"]))
        s["w"] = _kept(weights(N, K))
        s["bias"] = torch.randn(N, generator=g, device=dev) * 0.2 if case["bias"] else None
        s["residual"] = torch.randn((M, N), generator=g, device=dev).to(out) if case["residual"] else None
        s["out"] = torch.empty((M, N), dtype=out, device=dev)
        if own:
            from mlx_lm_b200 import ops
            s["codes"], s["scales"] = ops.fp8_empty(M, K, dev)
        return s

    T, E, top = case["tokens"], case["experts"], case["top"]
    s["logits"] = torch.randn((T, E), generator=g, device=dev) * 1.5
    s["correction"] = torch.randn(E, generator=g, device=dev) * 0.05 if case["correction"] else None
    # tokens of requests, and rows that pad the step
    s["req"] = torch.where(torch.rand(T, generator=g, device=dev) < case["live"], 0, -1).to(torch.int32)
    S = T * top
    s["sel"] = torch.empty(S, dtype=torch.int32, device=dev)
    s["weight"] = torch.empty(S, dtype=torch.float32, device=dev)
    s["sorted"] = torch.full((S,), -1, dtype=torch.int32, device=dev)
    if case["kind"] == "route":
        s["tile"] = case["tile"]
    if case["kind"] == "experts":
        D, F = case["width"], case["inner"]
        s["x"] = rows(T, D, torch.bfloat16)
        parts = [[weights(F, D), weights(F, D), weights(D, F)] for _ in range(E)]
        # gate rows, then up rows of every expert; its down rows
        s["w_in"] = _kept(torch.stack([torch.stack(p[:2]) for p in parts]))
        s["w_out"] = _kept(torch.stack([p[2] for p in parts]))
        s["out"] = torch.zeros((S, D), dtype=torch.bfloat16, device=dev)
        s["tile"] = 128
    if own:
        from mlx_lm_b200 import ops
        if case["kind"] == "experts":
            s["tile"] = ops.moe_fp8_tile_rows(S, E)
            most = ops.moe_max_tiles(S, E, s["tile"])
            s["codes"], s["scales"] = ops.fp8_empty(s["tile"], D, dev, groups=most)
            s["h_codes"], s["h_scales"] = ops.fp8_empty(s["tile"], F, dev, groups=most)
        s["scratch"] = torch.zeros(ops.moe_route_scratch(T, E), dtype=torch.int32, device=dev)
    most = -(-S // s["tile"]) + E
    s["tiles"] = torch.full((most, 3), -1, dtype=torch.int32, device=dev)
    s["n_tiles"] = torch.zeros(1, dtype=torch.int32, device=dev)
    return s


def _kept(w):
    """A weight as the program keeps it: codes with their scales (the framework lays them out), laid out once."""
    if own:
        from mlx_lm_b200 import ops
        R, K = w.shape[-2:]
        groups = w.numel() // (R * K)
        codes, scales = ops.fp8_empty(R, K, w.device, groups=groups)
        ops.fp8_quantize(w.view(-1, K), codes, scales, ops.current_stream(), group_rows=R)
        return codes, scales
    flat = w.view(-1, w.shape[-1])
    codes = torch.empty(flat.shape, dtype=torch.float8_e4m3fn, device=w.device)
    scales = torch.empty((flat.shape[0], -(-flat.shape[1] // BLOCK)), dtype=torch.float32, device=w.device)
    step = max(1, (1 << 26) // flat.shape[1])
    for a in range(0, flat.shape[0], step):
        codes[a:a + step], scales[a:a + step] = _quantize(flat[a:a + step])
    return codes.view(w.shape), scales.view(w.shape[:-1] + scales.shape[-1:])


# ------------------------------------------------------------------------------------------------ a pass

def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(state, kind)
    return _linear(state) if kind == "linear" else _experts(state) if kind == "experts" else _route(state)


def _own(s, kind):
    from mlx_lm_b200 import ops

    c, stream = s["case"], ops.current_stream()
    if kind == "linear":
        ops.fp8_quantize(s["x"], s["codes"], s["scales"], stream)
        ops.linear_fp8(s["codes"], s["scales"], *s["w"], s["bias"], s["out"], s["status"], stream, epilogue=ops.ACTIVATION_CODES[c["act"]],
                       residual=s["residual"])
        return dict(out=s["out"])
    E, top = c["experts"], c["top"]
    ops.moe_route_plan(s["logits"], s["req"], top, s["sel"], s["weight"], s["tile"], s["sorted"], s["tiles"], s["n_tiles"], s["scratch"],
                       stream, score=c["score"], renormalize=True, correction=s["correction"], groups=c["groups"], keep_groups=c["keep"],
                       group_score="two", weight_scale=SCALE)
    if kind == "route":
        return dict(expert=s["sel"], weight=s["weight"], order=s["sorted"], tiles=s["tiles"], n_tiles=s["n_tiles"])
    most = s["tiles"].shape[0]
    plan = (s["sorted"], s["tiles"], s["n_tiles"], most, s["tile"])
    ops.moe_gather_fp8(s["x"], top, *plan, s["codes"], s["scales"], stream)
    ops.moe_gemm_fp8(s["codes"], s["scales"], *s["w_in"], *plan, s["h_codes"], s["status"], stream, sel_weight=s["weight"], gated=True,
                     out_scales=s["h_scales"])
    ops.moe_gemm_fp8(s["h_codes"], s["h_scales"], *s["w_out"], *plan, s["out"], s["status"], stream)
    return dict(expert=s["sel"], weight=s["weight"], out=s["out"])


def _power(e):
    """``2**e`` in float32, exactly (a library's power need not be: half of the bfloat16 numbers next to a border lie on it)."""
    bits = torch.where(e > -127, (e + 127) << 23, 1 << 22)
    return bits.to(torch.int32).view(torch.float32)


def _quantize(x):
    """Rows to (codes, scales): the scale is a power of two, so that scaling is exact."""
    x = x.float()
    pad = -x.shape[1] % BLOCK
    b = torch.nn.functional.pad(x, (0, pad)).view(x.shape[0], -1, BLOCK)
    top = torch.where(torch.isfinite(b), b.abs(), 0.0).amax(-1)
    m, e = torch.frexp(top)                                  # top = m 2**e, m in [1/2, 1): 448 is 7/8 of 2**9
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(-127, 127)
    e = torch.where(top > 0, e, 0)
    scale = _power(e)
    codes = torch.where(torch.isfinite(b), b * _power(-e)[..., None], math.nan)
    return codes.view(x.shape[0], -1)[:, :x.shape[1]].to(torch.float8_e4m3fn), scale


def _values(codes, scale):
    x = codes.float()
    return x * scale.repeat_interleave(BLOCK, -1)[..., :x.shape[-1]]


def _held(x):
    return _values(*_quantize(x))


def _linear(s):
    c = s["case"]
    y = _held(s["x"]) @ _values(*s["w"]).T
    if s["bias"] is not None:
        y = y + s["bias"]
    if c["act"] == "relu":
        y = torch.clamp(y, min=0.0)
    elif c["act"] == "gelu_new":
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    s["out"].copy_(y)
    return dict(out=s["out"])


def _choose(s):
    """Choices and weights, in 64 bits: scores next to one another decide whole numbers."""
    c = s["case"]
    T, E, top, G = c["tokens"], c["experts"], c["top"], c["groups"]
    z = s["logits"].double()
    if c["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-z))
    else:
        e = torch.exp(z - z.amax(-1, keepdim=True))
        score = e / e.sum(-1, keepdim=True)
    by = score + s["correction"].double() if s["correction"] is not None else score
    if c["keep"] < G:
        two = by.view(T, G, E // G).sort(dim=-1, descending=True).values[..., :2].sum(-1)
        best = two.sort(dim=-1, descending=True, stable=True).indices[:, :c["keep"]]
        kept = torch.zeros((T, G), dtype=torch.bool, device=z.device).scatter(1, best, True)
        by = by.masked_fill(~kept.repeat_interleave(E // G, 1), -math.inf)
    sel = by.sort(dim=-1, descending=True, stable=True).indices[:, :top]
    w = score.gather(1, sel)
    w = w / w.sum(-1, keepdim=True) * SCALE
    live = (s["req"] >= 0)[:, None]
    s["sel"].copy_(torch.where(live, sel, -1).reshape(-1))
    s["weight"].copy_(torch.where(live, w, 0.0).reshape(-1))


def _route(s):
    c = s["case"]
    E, tile = c["experts"], c["tile"]
    _choose(s)
    sel = s["sel"].long()
    key = torch.where(sel >= 0, sel, E)
    order = key.sort(dim=0, stable=True).indices
    count = torch.zeros(E + 1, dtype=torch.long, device=sel.device).scatter_add(0, key, torch.ones_like(key))[:E]
    n = count.sum()
    place = torch.arange(sel.numel(), device=sel.device)
    s["sorted"].copy_(torch.where(place < n, order, s["sorted"].long()))
    first = count.cumsum(0) - count
    per = (count + tile - 1) // tile
    last = per.cumsum(0)
    i = torch.arange(s["tiles"].shape[0], device=sel.device)
    e = (i[:, None] >= last).sum(-1).clamp(max=E - 1)
    j = (i - (last - per)[e]) * tile
    made = torch.stack([e, first[e] + j, torch.clamp(count[e] - j, max=tile)], -1)
    s["tiles"].copy_(torch.where((i < last[-1])[:, None], made, s["tiles"].long()))
    s["n_tiles"].copy_(last[-1:])
    return dict(expert=s["sel"], weight=s["weight"], order=s["sorted"], tiles=s["tiles"], n_tiles=s["n_tiles"])


def _experts(s):
    c = s["case"]
    _choose(s)
    sel = s["sel"].long()
    x = _held(s["x"])
    order = sel.sort(dim=0, stable=True).indices
    counts = torch.zeros(c["experts"] + 1, dtype=torch.long, device=sel.device).scatter_add(0, sel + 1, torch.ones_like(sel)).tolist()
    at = counts[0]                                           # rows that pad the step come first
    for e in range(c["experts"]):
        n = counts[e + 1]
        if n == 0:
            continue
        slot = order[at:at + n]
        at += n
        rows, w = x[slot // c["top"]], s["weight"][slot][:, None]
        gate, up = (rows @ _values(s["w_in"][0][e, i], s["w_in"][1][e, i]).T for i in (0, 1))
        gate, up = w * gate, w * up
        h = _held(gate / (1.0 + torch.exp(-gate)) * up)
        s["out"][slot] = (h @ _values(s["w_out"][0][e], s["w_out"][1][e]).T).to(s["out"].dtype)
    return dict(expert=s["sel"], weight=s["weight"], out=s["out"])


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    item = dict(bfloat16=2, float32=4)
    if case["kind"] == "linear":
        M, K, N = case["rows"], case["inner"], case["outer"]
        nbytes = M * K * item[case["x"]] + N * K + N * -(-K // BLOCK) + M * N * item[case["out"]] * (2 if case["residual"] else 1)
        return dict(bytes=nbytes + (4 * N if case["bias"] else 0), flops=2 * M * N * K)
    T, E, top = case["tokens"], case["experts"], case["top"]
    S = T * top
    nbytes = 4 * T * E + 4 * T + 8 * S + (4 * E if case["correction"] else 0)
    if case["kind"] == "route":
        return dict(bytes=nbytes + 4 * S + 12 * min(S, S // case["tile"] + E), flops=8 * T * E)
    D, F = case["width"], case["inner"]
    live = int(T * case["live"])
    met = E * (1.0 - (1.0 - top / E) ** max(1, live))        # experts that some token chooses
    per = 2 * F * (D + -(-D // BLOCK)) + D * (F + -(-F // BLOCK))
    return dict(bytes=int(nbytes + live * (2 * D + top * 2 * D) + met * per), flops=6 * live * top * D * F)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits

def _exact_held(x):
    """What 8 bits hold of the rows of x, from the definition: scale and spacing of the codes by search."""
    x = x.double()
    K = x.shape[1]
    out = torch.empty_like(x)
    for a in range(0, K, BLOCK):
        b = x[:, a:a + BLOCK]
        top = b.abs().amax(1, keepdim=True)
        table = torch.tensor([math.ldexp(1.0, i) for i in range(-127, 128)], dtype=torch.float64, device=x.device)
        scale = table[torch.searchsorted(table * 448.0, top).clamp(max=254)]      # the first that reaches the largest magnitude
        v = b / torch.where(top > 0, scale, 1.0)
        spacing = table[127 - 6:127 + 9]                                          # 2**-6 .. 2**8: where the spacing of codes doubles
        step = spacing[(torch.searchsorted(spacing, v.abs(), right=True) - 1).clamp(min=0)] / 8.0
        out[:, a:a + BLOCK] = torch.round(v / step) * step * scale
    return out


def _exact_weight(kept):
    codes, scales = kept
    return codes.double() * scales.double().repeat_interleave(BLOCK, -1)[..., :codes.shape[-1]]


def exact(case, seed):
    global own
    before, own = own, False          # the plain layout of the weights, whoever asks
    try:
        s = prepare(case, seed)
    finally:
        own = before
    c = case
    if c["kind"] == "linear":
        y = _exact_held(s["x"]) @ _exact_weight(s["w"]).T
        if s["bias"] is not None:
            y += s["bias"].double()
        if c["act"] == "relu":
            y = torch.relu(y)
        elif c["act"] == "gelu_new":
            y = y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))
        if s["residual"] is not None:
            y += s["residual"].double()
        return dict(out=y)
    T, E, top, G = c["tokens"], c["experts"], c["top"], c["groups"]
    z = s["logits"].double()
    score = torch.sigmoid(z) if c["score"] == "sigmoid" else torch.softmax(z, -1)
    by = score + (s["correction"].double() if s["correction"] is not None else 0.0)
    if c["keep"] < G:
        groups = by.reshape(T, G, -1)
        order = groups.topk(2, -1).values.sum(-1).argsort(dim=-1, descending=True, stable=True)
        rank = order.argsort(-1)
        groups = torch.where((rank < c["keep"])[..., None], groups, -math.inf)
        by = groups.reshape(T, E)
    sel = by.argsort(dim=-1, descending=True, stable=True)[:, :top]
    w = torch.gather(score, 1, sel)
    w = w * (SCALE / w.sum(-1, keepdim=True))
    live = s["req"] >= 0
    sel[~live] = -1
    w[~live] = 0.0
    sel, w = sel.reshape(-1), w.reshape(-1)
    if c["kind"] == "route":
        order, tiles = s["sorted"].clone(), s["tiles"].clone()
        by_expert = [[] for _ in range(E)]
        for slot, e in enumerate(sel.tolist()):
            if e >= 0:
                by_expert[e].append(slot)
        flat, made = [], []
        for e, slots in enumerate(by_expert):
            made += [(e, len(flat) + a, min(c["tile"], len(slots) - a)) for a in range(0, len(slots), c["tile"])]
            flat += slots
        if made:
            order[:len(flat)] = torch.tensor(flat, dtype=torch.int32, device=order.device)
            tiles[:len(made)] = torch.tensor(made, dtype=torch.int32, device=order.device)
        n = torch.tensor([len(made)], dtype=torch.int32, device=order.device)
        return dict(expert=sel.to(torch.int32), weight=w, order=order, tiles=tiles, n_tiles=n)
    x = _exact_held(s["x"])
    y = torch.zeros((T * top, c["width"]), dtype=torch.float64, device=x.device)
    for e in range(E):
        slots = torch.nonzero(sel == e).view(-1)
        if slots.numel() == 0:
            continue
        rows = x[torch.div(slots, top, rounding_mode="floor")] * w[slots, None].float().double()
        gate = rows @ _exact_weight((s["w_in"][0][e, 0], s["w_in"][1][e, 0])).T
        up = rows @ _exact_weight((s["w_in"][0][e, 1], s["w_in"][1][e, 1])).T
        h = _exact_held(gate * torch.sigmoid(gate) * up)
        y[slots] = h @ _exact_weight((s["w_out"][0][e], s["w_out"][1][e])).T
    return dict(expert=sel.to(torch.int32), weight=w, out=y)
