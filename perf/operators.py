"""Operators of a paged key/value cache that is held in 8 bits, as cases that can be timed and compared.

A page holds ``page`` positions of every key/value head as int8 codes ``[n_pages, heads, page, head_dim]``; every block of 16
positions of a head has one float32 scale ``[n_pages, heads, page // 16]``, and a code stands for ``code * scale``.

``append``    a step's keys and values enter the pages, keys (and the queries beside them) turned by their position on the way,
              then the blocks that the step touched are read back: outputs are the turned queries, the values that the cache now
              stands for in these blocks, and all scales.  Both are what a program does that keeps such a cache: a step writes it,
              and a cache that is saved or looked at is read.
``rows``      attention of one query a request over its pages: decode steps.
``portions``  attention of runs of queries of each request over its pages: prompts that arrive whole or in portions.

What an append does to a block: ``A`` is the largest magnitude among the finite numbers it brings for a head, ``S = A / 127`` (0 below
2**-100).  If the append brings the block's first position the scale becomes ``S``, else the larger of ``S`` and the old scale; if the
scale grows, the older codes become ``rint(code * (old / new))``.  New codes are ``rint(x * (1 / scale))`` within -127 .. 127.

Sizes: heads of the configurations of this repository (12, 16, 20 and 25 heads of 64, grouped heads of 48 and 64) and generic grouped
ones (of 96 and 128); pages of 16 to 128 positions; 1 to 64 requests; contexts of 1 to 131072 positions; up to 8192 tokens a step.
"""
import math

import torch

own = False

BLOCK = 16


# ------------------------------------------------------------------------------------------------ the cases

def listed():
    return [
        # one user's chat: a single token enters the cache in the middle of a block; launches are all of it
        dict(name="append 1", kind="append", dtype="bfloat16", heads=32, kv_heads=8, dim=128, rot=128, page=16, requests=1, tokens=1,
             context=517, ragged=False),
        # a full batch of requests, one token each, every one at a place of its own in its block
        dict(name="append 64 rows", kind="append", dtype="bfloat16", heads=32, kv_heads=8, dim=128, rot=128, page=16, requests=64, tokens=1,
             context=4096, ragged=True),
        # prompts of GPT-2 size in the 32-bit path: no rotation, portions that begin and end inside a block
        dict(name="append ragged float32", kind="append", dtype="float32", heads=16, kv_heads=16, dim=64, rot=0, page=16, requests=5,
             tokens=331, context=100, ragged=True),
        # a long document in one step
        dict(name="append 8192", kind="append", dtype="bfloat16", heads=32, kv_heads=8, dim=128, rot=128, page=64, requests=1, tokens=8192,
             context=0, ragged=False),
        # one user's chat with GPT-2 medium
        dict(name="rows 1 of 16x64", kind="rows", dtype="bfloat16", heads=16, kv_heads=16, dim=64, page=16, requests=1, context=520,
             window=0, sinks=False, ragged=False),
        # a few users with grouped heads, lengths of their own
        dict(name="rows 8 of 32/8x128", kind="rows", dtype="bfloat16", heads=32, kv_heads=8, dim=128, page=16, requests=8, context=4000,
             window=0, sinks=False, ragged=True),
        # a full batch at long contexts
        dict(name="rows 64 of 32/8x128", kind="rows", dtype="bfloat16", heads=32, kv_heads=8, dim=128, page=16, requests=64, context=8192,
             window=0, sinks=False, ragged=True),
        # one very long document
        dict(name="rows 1 at 131072", kind="rows", dtype="bfloat16", heads=32, kv_heads=8, dim=128, page=64, requests=1, context=131072,
             window=0, sinks=False, ragged=False),
        # the 32-bit path: a window and sinks, few requests
        dict(name="rows window float32", kind="rows", dtype="float32", heads=16, kv_heads=4, dim=64, page=16, requests=4, context=3001,
             window=1000, sinks=True, ragged=True),
        # a short turn of a chat behind a cached one: grouped heads of 48, a window, sinks
        dict(name="portion 77 of 6/3x48", kind="portions", dtype="bfloat16", heads=6, kv_heads=3, dim=48, page=16, requests=1, tokens=77,
             context=900, window=600, sinks=True, ragged=False),
        # two whole prompts of GPT-2 medium
        dict(name="portions 2x1024 of 16x64", kind="portions", dtype="bfloat16", heads=16, kv_heads=16, dim=64, page=16, requests=2,
             tokens=1024, context=0, window=0, sinks=False, ragged=False),
        # the last portion of a long document, grouped heads
        dict(name="portion 2048 at 6144", kind="portions", dtype="bfloat16", heads=32, kv_heads=8, dim=128, page=16, requests=1, tokens=2048,
             context=6144, window=0, sinks=False, ragged=False),
    ]


HEADS = [(12, 12, 64), (16, 16, 64), (20, 20, 64), (25, 25, 64), (6, 3, 48), (16, 4, 64), (16, 4, 96), (8, 2, 128), (16, 2, 128),
         (32, 8, 128), (64, 8, 128)]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "rows", "rows", "portions"])
    heads, kv_heads, dim = rng.choice(HEADS)
    case = dict(kind=kind, dtype="float32" if kind != "portions" and rng.random() < 0.15 else "bfloat16", heads=heads, kv_heads=kv_heads,
                dim=dim, page=rng.choice([16, 16, 32, 64, 128]), ragged=rng.random() < 0.7)
    if kind == "append":
        case["rot"] = rng.choice([0, dim // 2, dim])
        case["requests"] = _spread(rng, 1, 64)
        case["tokens"] = 1 if rng.random() < 0.4 else _spread(rng, 1, max(1, 8192 // case["requests"]))
        case["context"] = _spread(rng, 1, 4096) - 1
        if heads == 64:
            case["tokens"] = min(case["tokens"], max(1, 4096 // case["requests"]))
    elif kind == "rows":
        case["requests"] = _spread(rng, 1, 64)
        most = (64 * 8192 * 8 * 128) // (case["requests"] * kv_heads * dim)
        if case["dtype"] == "float32":
            most //= 16
        case["context"] = _spread(rng, 1, min(131072, most))
        case["window"] = _spread(rng, 1, case["context"]) if rng.random() < 0.25 else 0
        case["sinks"] = rng.random() < 0.25
    else:
        case["requests"] = _spread(rng, 1, 4)
        case["tokens"] = _spread(rng, 2, 2048 // case["requests"])
        case["context"] = _spread(rng, 1, 6144) - 1
        if heads == 64:
            case["tokens"] = min(case["tokens"], max(2, 1024 // case["requests"]))
        case["window"] = _spread(rng, 1, case["context"] + case["tokens"]) if rng.random() < 0.25 else 0
        case["sinks"] = rng.random() < 0.25
    return case


def _lengths(case):
    """``[(positions that a request holds before, tokens that it brings)]``: the same for every seed, ragged ones all different."""
    n, out = case["requests"], []
    for i in range(n):
        share = 1.0 if not case["ragged"] or i == 0 else (1 + (i * 37) % 64) / 64.0
        if case["kind"] == "rows":
            out.append((max(1, int(case["context"] * share)) - 1, 1))
        else:
            tokens = case["tokens"] if case["tokens"] == 1 else max(1, int(case["tokens"] * share))
            out.append((int(case["context"] * share), tokens))
    return out


# ------------------------------------------------------------------------------------------------ inputs

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    H, G, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    lengths = _lengths(case)
    n_req = len(lengths)
    need = [-(-(c + t) // page) for c, t in lengths]
    width = max(need)
    n_pages = sum(need) + 3
    ids = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((n_req, width), -1, dtype=torch.int32)
    for r, n in enumerate(need):
        table[r, :n] = torch.tensor(ids[:n], dtype=torch.int32)
        ids = ids[n:]
    pos = torch.cat([torch.arange(c, c + t, dtype=torch.int32) for c, t in lengths])
    req = torch.cat([torch.full((t,), r, dtype=torch.int32) for r, (c, t) in enumerate(lengths)])
    T = pos.numel()

    def codes():
        # what rounding normal numbers to a block's largest magnitude leaves: a spread of about 127 / 3.3
        x = torch.empty((n_pages, G, page, D), dtype=torch.bfloat16, device=dev).normal_(0.0, 38.0, generator=g)
        return x.round_().clamp_(-127, 127).to(torch.int8)

    def scales(size):
        return torch.empty((n_pages, G, page // BLOCK), dtype=torch.float32, device=dev).uniform_(0.7, 1.4, generator=g).mul_(size / 38.0)

    def normal(*shape, size=1.0):
        return (torch.randn(shape, generator=g, device=dev) * size).to(dtype)

    s = dict(case=case, table=table.to(dev), pos=pos.to(dev), req=req.to(dev), k8=codes(), v8=codes(), ks=scales(1.0), vs=scales(0.7),
             status=torch.zeros(1, dtype=torch.int32, device=dev), lengths=lengths, longest=max(c + t for c, t in lengths))
    if case["kind"] == "append":
        # one fused projection a token, as layers make it: queries, keys and values are columns of the same rows.  Some columns of
        # keys are much larger than others.
        size = torch.ones((H + 2 * G) * D, device=dev)
        size[H * D:(H + G) * D:17] = 6.0
        s["qkv"] = (torch.randn((T, (H + 2 * G) * D), generator=g, device=dev) * size).to(dtype)
        s["q_out"] = torch.empty((T, H * D), dtype=dtype, device=dev)
        if case["rot"]:
            i = torch.arange(case["rot"] // 2, dtype=torch.float64)
            s["freq"] = (10000.0 ** (-2.0 * i / case["rot"])).to(torch.float32).to(dev)
        else:
            s["freq"] = None
        # every position of the blocks that the step touches, up to the last that holds something
        rp = [torch.arange(c // BLOCK * BLOCK, c + t, dtype=torch.int32) for c, t in lengths]
        s["read_pos"] = torch.cat(rp).to(dev)
        s["read_req"] = torch.cat([torch.full((x.numel(),), r, dtype=torch.int32) for r, x in enumerate(rp)]).to(dev)
        s["touched_pos"] = torch.cat([x[::BLOCK] for x in rp]).to(dev)
        s["touched_req"] = torch.cat([torch.full((x[::BLOCK].numel(),), r, dtype=torch.int32) for r, x in enumerate(rp)]).to(dev)
        s["k_read"] = torch.empty((s["read_pos"].numel(), G * D), dtype=dtype, device=dev)
        s["v_read"] = torch.empty_like(s["k_read"])
    else:
        s["q"] = normal(T, H * D, size=2.0)
        s["out"] = torch.empty((T, H * D), dtype=dtype, device=dev)
        s["scale"] = D ** -0.5
        s["sinks"] = torch.randn(H, generator=g, device=dev) if case["sinks"] else None
    if case["kind"] == "portions":
        tiles, row, at = [], 0, []
        most = max(t for c, t in lengths)
        for r, (c, t) in enumerate(lengths):
            tiles += [(row + a, min(128, t - a), r, c + a) for a in range(0, t, 128)]
            at.append(torch.cat([torch.arange(row, row + t), torch.full((most - t,), -1)]))
            row += t
        tiles.sort(key=lambda x: -(x[1] + x[3]))
        s["tiles"] = torch.tensor(tiles, dtype=torch.int32, device=dev)
        s["at"] = torch.stack(at).to(dev)                  # rows of each request's queries, -1 behind its last
        s["first"] = torch.tensor([c for c, t in lengths], dtype=torch.int32, device=dev)
    return s


# ------------------------------------------------------------------------------------------------ a pass

def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(state, kind)
    return _append(state) if kind == "append" else _rows(state) if kind == "rows" else _portions(state)


def _own(s, kind):
    from mlx_lm_b200 import ops

    c, stream = s["case"], ops.current_stream()
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    if kind == "append":
        q, k, v = (s["qkv"][:, a * D:b * D] for a, b in ((0, H), (H, H + G), (H + G, H + 2 * G)))
        ops.kv8_append(k, v, s["pos"], s["req"], s["table"], s["k8"], s["v8"], s["ks"], s["vs"], s["status"], stream, freq=s["freq"],
                       q=q, q_out=s["q_out"])
        ops.kv8_read(s["read_pos"], s["read_req"], s["table"], s["k8"], s["v8"], s["ks"], s["vs"], s["k_read"], s["v_read"], s["status"],
                     stream)
        return dict(q=s["q_out"], k=s["k_read"], v=s["v_read"], k_scale=s["ks"], v_scale=s["vs"])
    if kind == "rows":
        if "scratch" not in s:      # kept by the program from step to step
            floats, tickets = ops.kv8_rows_scratch(s["q"].shape[0], H, G, D, s["longest"])
            s["scratch"] = torch.zeros(floats, dtype=torch.float32, device=s["q"].device)
            s["tickets"] = torch.zeros(tickets, dtype=torch.int32, device=s["q"].device)
        ops.kv8_attention_rows(s["q"], s["pos"], s["req"], s["table"], s["k8"], s["v8"], s["ks"], s["vs"], s["out"], H, s["scale"],
                               c["window"], s["scratch"], s["tickets"], s["longest"], s["status"], stream, sinks=s["sinks"])
    else:
        ops.kv8_attention_portions(s["q"], s["tiles"], s["tiles"].shape[0], s["table"], s["k8"], s["v8"], s["ks"], s["vs"], s["out"], H,
                                   s["scale"], c["window"], s["status"], stream, sinks=s["sinks"])
    return dict(out=s["out"])


def _turn(x, pos, freq):
    """``x [T, heads, dim]`` float32: the first ``2 * len(freq)`` dimensions turn, pairs ``(i, i + len(freq))``."""
    if freq is None:
        return x
    h = freq.numel()
    a = pos.to(torch.float32)[:, None] * freq
    c, s = torch.cos(a)[:, None], torch.sin(a)[:, None]
    u, v = x[..., :h], x[..., h:2 * h]
    return torch.cat([u * c - v * s, v * c + u * s, x[..., 2 * h:]], -1)


def _enter(s, x, pool, scale):
    """Rows ``x [T, heads, dim]`` into the pages."""
    pos, req, page = s["pos"].long(), s["req"].long(), s["case"]["page"]
    per = page // BLOCK
    pg = s["table"].long()[req, pos // page]
    block = pg * per + pos % page // BLOCK                 # of all blocks of the pool
    n = scale.shape[0] * per
    heads = x.shape[1]
    fine = torch.isfinite(x)
    top = torch.where(fine, x.abs(), 0.0).amax(-1)
    largest = torch.zeros((n, heads), device=x.device).scatter_reduce(0, block[:, None].expand(-1, heads), top, "amax")
    opened = torch.zeros(n, dtype=torch.bool, device=x.device).index_fill(0, torch.where(pos % BLOCK == 0, block, block[0]), True)
    opened[block[0]] = pos[0] % BLOCK == 0                 # (rows inside a block stood for the first row's)
    tp, tr = s["touched_pos"].long(), s["touched_req"].long()
    tpg, tsub = s["table"].long()[tr, tp // page], tp % page // BLOCK
    t = tpg * per + tsub
    old = scale[tpg, :, tsub]
    new = torch.where(largest[t] < 2.0 ** -100, 0.0, largest[t] / 127.0)
    new = torch.where(opened[t][:, None], new, torch.maximum(old, new))
    view = pool.view(pool.shape[0], heads, per, BLOCK, pool.shape[3])
    kept = view[tpg, :, tsub].float()
    grown = ((new > old) & ~opened[t][:, None])[..., None, None]
    ratio = (old / torch.where(new > 0, new, 1.0))[..., None, None]
    view[tpg, :, tsub] = torch.where(grown, torch.round(kept * ratio), kept).to(torch.int8)
    scale[tpg, :, tsub] = new
    now = scale[pg, :, pos % page // BLOCK][..., None]
    inv = torch.where(now > 0, 1.0 / now, 0.0)
    code = torch.where(torch.isnan(x), 0.0, torch.round(x * inv).clamp(-127, 127))
    pool[pg, :, pos % page] = torch.where(now > 0, code, 0.0).to(torch.int8)


def _append(s):
    c = s["case"]
    H, G, D, T, page = c["heads"], c["kv_heads"], c["dim"], s["pos"].numel(), c["page"]
    x = s["qkv"].float().view(T, H + 2 * G, D)
    s["q_out"].copy_(_turn(x[:, :H], s["pos"], s["freq"]).reshape(T, H * D))
    _enter(s, _turn(x[:, H:H + G], s["pos"], s["freq"]), s["k8"], s["ks"])
    _enter(s, x[:, H + G:], s["v8"], s["vs"])
    rp, rr = s["read_pos"].long(), s["read_req"].long()
    pg, sub, at = s["table"].long()[rr, rp // page], rp % page // BLOCK, rp % page
    s["k_read"].copy_((s["k8"][pg, :, at].float() * s["ks"][pg, :, sub][..., None]).reshape(-1, G * D))
    s["v_read"].copy_((s["v8"][pg, :, at].float() * s["vs"][pg, :, sub][..., None]).reshape(-1, G * D))
    return dict(q=s["q_out"], k=s["k_read"], v=s["v_read"], k_scale=s["ks"], v_scale=s["vs"])


def _held(s, pool, scale):
    """``[requests, heads, longest, dim]`` float32: what the pages stand for (positions without a page: some other page's)."""
    page, n = s["case"]["page"], s["longest"]
    j = torch.arange(n, device=pool.device)
    pg = s["table"].long()[:, j // page].clamp(min=0)
    x = pool[pg, :, j % page].float() * scale[pg, :, j % page // BLOCK][..., None]        # [requests, n, heads, dim]
    return x.transpose(1, 2)


def _attend(q, k, v, p, scale, window, sinks):
    """``q [R, G, g, n, D]`` at positions ``p [R, n]`` over ``k, v [R, G, L, D]``."""
    R, G, g, n, D = q.shape
    x = (q.reshape(R, G, g * n, D) @ k.transpose(-1, -2)).view(R, G, g, n, -1) * scale
    j = torch.arange(k.shape[2], device=q.device)
    seen = j <= p[..., None]
    if window:
        seen &= j > p[..., None] - window
    x = x.masked_fill(~seen[:, None, None], float("-inf"))
    m = x.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), 0.0, m)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    y = (e.view(R, G, g * n, -1) @ v).view(R, G, g, n, D)
    if sinks is not None:
        total = total + torch.exp(sinks.view(1, G, g, 1, 1) - m)
    return y / total


def _rows(s):
    c = s["case"]
    R, H, G, D = s["pos"].numel(), c["heads"], c["kv_heads"], c["dim"]
    q = s["q"].float().view(R, G, H // G, 1, D)
    y = _attend(q, _held(s, s["k8"], s["ks"]), _held(s, s["v8"], s["vs"]), s["pos"][:, None], s["scale"], c["window"], s["sinks"])
    s["out"].copy_(y.reshape(R, H * D))
    return dict(out=s["out"])


def _portions(s):
    c = s["case"]
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    at = s["at"]
    R, n = at.shape
    q = s["q"].float()[at.clamp(min=0)].view(R, n, G, H // G, D).permute(0, 2, 3, 1, 4)
    p = s["first"][:, None] + torch.arange(n, device=q.device)
    y = _attend(q, _held(s, s["k8"], s["ks"]), _held(s, s["v8"], s["vs"]), p, s["scale"], c["window"], s["sinks"])
    y = y.permute(0, 3, 1, 2, 4).reshape(R, n, H * D)
    s["out"][at[at >= 0]] = y[at >= 0].to(s["out"].dtype)
    return dict(out=s["out"])


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    item = 4 if case["dtype"] == "float32" else 2
    lengths = _lengths(case)
    T = sum(t for c, t in lengths)
    if case["kind"] == "append":
        touched = sum(c + t - c // BLOCK * BLOCK for c, t in lengths)
        blocks = sum(-(-(c + t) // BLOCK) - c // BLOCK for c, t in lengths)
        nbytes = T * (2 * H + 2 * G) * D * item + T * 2 * G * D + blocks * 2 * G * 8 + touched * 2 * G * D * (1 + item)
        return dict(bytes=nbytes, flops=T * D * (3 * H + 8 * G))
    window = case["window"]
    keys = pairs = blocks = 0
    for c, t in lengths:
        first = max(0, c - window + 1) if window else 0
        keys += c + t - first
        blocks += -(-(c + t) // BLOCK) - first // BLOCK
        if window:
            pairs += sum(min(window, p + 1) for p in range(c, c + t))
        else:
            pairs += t * c + t * (t + 1) // 2
    return dict(bytes=keys * 2 * G * D + blocks * 2 * G * 4 + 2 * T * H * D * item, flops=4 * H * D * pairs)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    H, G, D, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    per = page // BLOCK

    def pages(pool, scale, r, first, last):
        """``[heads, last - first, dim]`` in 64 bits: positions ``first .. last - 1`` of request r."""
        a, b = first // page, -(-last // page)
        ids = s["table"][r, a:b].long()
        x = pool[ids].double() * scale[ids].double().repeat_interleave(BLOCK, 2)[..., None]
        x = x.permute(1, 0, 2, 3).reshape(pool.shape[1], -1, pool.shape[3])
        return x[:, first - a * page:last - a * page]

    if c["kind"] != "append":
        y = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        row = 0
        for r, (before, t) in enumerate(s["lengths"]):
            lo = max(0, before - c["window"] + 1) if c["window"] else 0
            k, v = pages(s["k8"], s["ks"], r, lo, before + t), pages(s["v8"], s["vs"], r, lo, before + t)
            q = s["q"][row:row + t].double().view(t, H, D)
            i = torch.arange(before, before + t, device=q.device)[:, None]
            j = torch.arange(lo, before + t, device=q.device)[None]
            hidden = (j > i) | ((i - j >= c["window"]) if c["window"] else (j < 0))
            for h in range(H):
                x = (q[:, h] @ k[h // (H // G)].T) * s["scale"]
                x[hidden] = -math.inf
                if s["sinks"] is not None:
                    x = torch.cat([x, s["sinks"][h].double().expand(t, 1)], 1)
                y[row:row + t, h * D:(h + 1) * D] = torch.softmax(x, 1)[:, :k.shape[1]] @ v[h // (H // G)]
            row += t
        return dict(out=y)

    T = s["pos"].numel()
    x = s["qkv"].double().view(T, H + 2 * G, D).clone()
    if s["freq"] is not None:
        h = s["freq"].numel()
        angle = (s["pos"].float()[:, None] * s["freq"]).double()[:, None]      # the angle itself is a 32-bit number
        z = torch.polar(torch.ones_like(angle), angle) * torch.complex(x[:, :H + G, :h], x[:, :H + G, h:2 * h])
        x[:, :H + G, :h], x[:, :H + G, h:2 * h] = z.real, z.imag
    got = dict(q=x[:, :H].reshape(T, H * D))
    for name, pool, scale, rows in (("k", s["k8"], s["ks"], x[:, H:H + G]), ("v", s["v8"], s["vs"], x[:, H + G:])):
        scales, out, row = scale.double(), [], 0
        for r, (before, t) in enumerate(s["lengths"]):
            a = before // BLOCK * BLOCK
            n = before + t - a
            blocks = -(-n // BLOCK)
            held = torch.zeros((G, blocks * BLOCK, D), dtype=torch.float64, device=x.device)
            new = torch.zeros_like(held)
            new[:, before - a:n] = rows[row:row + t].transpose(0, 1)
            logical = torch.arange(a, a + blocks * BLOCK, BLOCK, device=x.device)
            ids, sub = s["table"][r].long()[logical // page], logical % page // BLOCK
            size = new.view(G, blocks, BLOCK * D).abs().amax(2) / 127
            if before > a:          # the first block holds older tokens
                old = scales[ids[0], :, sub[0]]
                size[:, 0] = torch.maximum(size[:, 0], old)
                w = int(sub[0]) * BLOCK
                codes = pool[ids[0], :, w:w + before - a].double()
                held[:, :before - a] = torch.round(codes * (old / size[:, 0])[:, None, None]) * size[:, 0][:, None, None]
            wide = size.repeat_interleave(BLOCK, 1)[..., None]
            entered = torch.round(new / wide).clamp(-127, 127) * wide
            held[:, before - a:n] = entered[:, before - a:n]
            scales[ids, :, sub] = size.T
            out.append(held[:, :n].transpose(0, 1).reshape(n, G * D))
            row += t
        got[name], got[name + "_scale"] = torch.cat(out), scales
    return got
