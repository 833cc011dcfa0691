"""The order of kernels on a stream: a launch that has nothing to do still ends after the one before it, so that the one behind it sees
what that has written."""
import pytest
import torch

import kv8_refs as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("between", ["append", "portions of nothing", "portions out of range"])
def test_a_launch_with_nothing_to_do_keeps_the_order(between):
    from mlx_lm_b200 import ops
    heads, dim, page, n = 8, 128, 16, 8192
    cache = R.Cache([n], heads, dim, page, seed=1, filled=False)
    dev, table = cache.cuda(), cache.table.cuda()
    pos, req = (t.cuda() for t in R.steps([(0, n)]))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    few, nobody = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.full((4,), -1, dtype=torch.int32, device="cuda")
    q = torch.zeros(4, heads * dim, dtype=torch.bfloat16, device="cuda")
    tiles = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    if between == "portions out of range":
        tiles[:, 1], tiles[:, 2] = 1, 7
    last = torch.arange(n - 64, n, dtype=torch.int32, device="cuda")
    owner = torch.zeros(64, dtype=torch.int32, device="cuda")
    stream = ops.current_stream()

    def nothing():
        if between == "append":
            ops.kv8_append(q, q, few, nobody, table, *dev, status, stream)
        else:
            ops.kv8_attention_portions(q, tiles, 2, table, *dev, torch.empty_like(q), heads, 0.1, 0, status, stream)

    nothing()                                     # (its library is loaded before the order matters)
    for i in range(20):
        x = torch.full((n, heads * dim), float(i + 1), dtype=torch.bfloat16, device="cuda")
        k, v = torch.zeros(64, heads * dim, device="cuda"), torch.zeros(64, heads * dim, device="cuda")
        torch.cuda.synchronize()
        ops.kv8_append(x, x, pos, req, table, *dev, status, stream)
        nothing()
        ops.kv8_read(last, owner, table, *dev, k, v, status, stream)
        # one number everywhere: the code 127 of a scale of (i + 1) / 127, each of the two roundings 2**-24 of the number
        for got in (k, v):
            assert float((got - (i + 1)).abs().max()) <= (i + 1) * 2.0 ** -22
    assert int(status.item()) == (ops.ST_POSITION_RANGE if between == "portions out of range" else 0)


def test_tiles_start_in_the_order_of_their_list():
    """One tile of many keys and as much work in short tiles: with the long one first they run beside one another, with it last they add
    up.  (Blocks start in the order of their numbers; the least of several times, and a wide margin.)"""
    from mlx_lm_b200 import ops
    heads, dim, page, long, short, n = 16, 64, 128, 16384, 0, 650
    g = torch.Generator(device="cuda").manual_seed(1)
    n_pages = long // page + 2
    k8, v8 = (torch.randint(-127, 128, (n_pages, heads, page, dim), generator=g, device="cuda", dtype=torch.int32).to(torch.int8) for _ in range(2))
    ks, vs = (torch.full((n_pages, heads, page // 16), 0.01, device="cuda") for _ in range(2))
    table = torch.arange(n_pages, dtype=torch.int32, device="cuda").view(1, -1)
    q = torch.randn((n + 1) * 128, heads * dim, generator=g, device="cuda").bfloat16()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    tiles = [(0, 128, 0, long)] + [(128 * (i + 1), 128, 0, short) for i in range(n)]

    def run(order):
        t, out, best = torch.tensor(order, dtype=torch.int32, device="cuda"), torch.empty_like(q), float("inf")
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            a.record()
            ops.kv8_attention_portions(q, t, len(order), table, k8, v8, ks, vs, out, heads, 0.125, 0, status, ops.current_stream())
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best, out

    (first, out), (last, same) = run(tiles), run(tiles[::-1])
    assert int(status.item()) == 0 and torch.equal(out, same)
    print(f"the long tile first {first * 1e3:.0f} us, last {last * 1e3:.0f} us")
    assert first < 0.8 * last
