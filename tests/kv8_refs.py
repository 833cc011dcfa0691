"""Plain statements, on the CPU, of the operators of a key/value cache in 8 bits: appends in float32 with every rounding where the
kernel has it, what the pages stand for and attention over them in float64.  Nothing here is imported by the package."""
import math

import torch

BLOCK = 16


class Cache:
    """Pages of one layer with a block table in scrambled order, on the CPU."""

    def __init__(self, lengths, heads, dim, page, seed, spare=2, filled=True):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.dim, self.page = heads, dim, page
        need = [-(-n // page) for n in lengths]
        width = max(need) + 1
        n_pages = sum(need) + spare
        ids = torch.randperm(n_pages, generator=g).tolist()
        self.table = torch.full((len(lengths), width), -1, dtype=torch.int32)
        for r, n in enumerate(need):
            self.table[r, :n] = torch.tensor(ids[:n], dtype=torch.int32)
            ids = ids[n:]
        shape = (n_pages, heads, page, dim)
        self.k8, self.v8 = (torch.randint(-127, 128, shape, generator=g, dtype=torch.int32).to(torch.int8) for _ in range(2))
        self.ks, self.vs = (torch.rand((n_pages, heads, page // BLOCK), generator=g) * 0.02 + 0.005 for _ in range(2))
        if not filled:
            for t in (self.k8, self.v8, self.ks, self.vs):
                t.zero_()

    def tensors(self):
        return self.k8, self.v8, self.ks, self.vs

    def cuda(self):
        return [t.cuda() for t in self.tensors()]

    def held(self, pool, scale, r, first, last):
        """float64 ``[heads, last - first, dim]``: positions ``first .. last - 1`` of request r."""
        out = []
        for p in range(first, last):
            pg = int(self.table[r, p // self.page])
            assert pg >= 0, f"position {p} has no page"
            at = p % self.page
            out.append(pool[pg, :, at].double() * scale[pg, :, at // BLOCK, None].double())
        return torch.stack(out, 1)


def turn(x, positions, freq, interleaved=False, mscale=1.0):
    """float32 ``x [T, heads, dim]``, every product and sum rounded by itself."""
    if freq is None or not freq.numel():
        return x.clone()
    h = freq.numel()
    a = positions.float()[:, None] * freq
    c = (torch.cos(a.double()).float() * mscale)[:, None]
    s = (torch.sin(a.double()).float() * mscale)[:, None]
    y = x.clone()
    if interleaved:
        u, v = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
        y[..., 0:2 * h:2], y[..., 1:2 * h:2] = u * c - v * s, v * c + u * s
    else:
        u, v = x[..., :h], x[..., h:2 * h]
        y[..., :h], y[..., h:2 * h] = u * c - v * s, v * c + u * s
    return y


def enter(cache, pool, scale, x, positions, token_req):
    """Rows ``x [T, heads, dim]`` (float32) into ``pool`` and ``scale``, in place."""
    T = x.shape[0]
    t = 0
    while t < T:
        r = int(token_req[t])
        if r < 0:
            t += 1
            continue
        p = int(positions[t])
        n = 1
        while (t + n < T and int(token_req[t + n]) == r and int(positions[t + n]) == p + n and (p + n) % BLOCK):
            n += 1
        pg = int(cache.table[r, p // cache.page])
        if pg >= 0:
            rows = x[t:t + n]
            fine = torch.isfinite(rows)
            top = torch.where(fine, rows.abs(), torch.zeros(())).amax((0, 2))
            new = torch.where(top < 2.0 ** -100, torch.zeros(()), top / 127.0)
            at, sub, off = p % cache.page, p % cache.page // BLOCK, p % BLOCK
            if off:
                old = scale[pg, :, sub].clone()
                for h in range(cache.heads):
                    if new[h] > old[h]:
                        old_codes = pool[pg, h, at - off:at].float()
                        pool[pg, h, at - off:at] = torch.round(old_codes * (old[h] / new[h])).to(torch.int8)
                new = torch.maximum(old, new)
            scale[pg, :, sub] = new
            inv = torch.where(new > 0, 1.0 / new, torch.zeros(()))
            codes = torch.where(torch.isnan(rows), torch.zeros(()), torch.round(rows * inv[None, :, None]).clamp(-127, 127))
            codes = torch.where((new > 0)[None, :, None], codes, torch.zeros(()))
            pool[pg, :, at:at + n] = codes.to(torch.int8).transpose(0, 1)
        t += n


def attention(cache, q, positions, token_req, n_heads, scale, window=0, sinks=None):
    """float64 ``[T, n_heads * dim]``; rows of no request are zeros."""
    T, G, D = q.shape[0], cache.heads, cache.dim
    out = torch.zeros(T, n_heads, D, dtype=torch.float64)
    rep = n_heads // G
    kept = {}
    for t in range(T):
        r = int(token_req[t])
        if r < 0:
            continue
        last = max(int(positions[i]) for i in range(T) if int(token_req[i]) == r) + 1
        if r not in kept:
            lo = min(max(0, int(positions[i]) - window + 1) if window else 0 for i in range(T) if int(token_req[i]) == r)
            kept[r] = (lo, cache.held(cache.k8, cache.ks, r, lo, last), cache.held(cache.v8, cache.vs, r, lo, last))
        base, k, v = kept[r]
        p = int(positions[t])
        lo = max(0, p - window + 1) if window else 0
        kk = k[:, lo - base:p + 1 - base].repeat_interleave(rep, 0)
        vv = v[:, lo - base:p + 1 - base].repeat_interleave(rep, 0)
        s = torch.einsum("hd,hnd->hn", q[t].double().view(n_heads, D), kk) * scale
        if sinks is not None:
            s = torch.cat([s, sinks.double()[:, None]], 1)
        w = torch.softmax(s, 1)[:, :kk.shape[1]]
        out[t] = torch.einsum("hn,hnd->hd", w, vv)
    return out.view(T, n_heads * D)


def steps(spans):
    """``(positions, token_req)`` of requests that bring ``[(first position, tokens)]``."""
    pos = torch.cat([torch.arange(a, a + n, dtype=torch.int32) for a, n in spans])
    req = torch.cat([torch.full((n,), r, dtype=torch.int32) for r, (a, n) in enumerate(spans)])
    return pos, req


def frequencies(half, base=10000.0):
    return (base ** (-torch.arange(half, dtype=torch.float64) / max(1, half))).float()
