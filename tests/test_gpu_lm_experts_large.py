"""Routing, expert products, their combination and clipping over arrays of more than 2^31 elements: the rows at the end against the
same rows by themselves, or against 64 bits."""
import pytest
import torch

import lm_expert_reference as er
import lm_reference as ref
import stquant_lm as lm

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def big(rows, width, dtype, seed, std=1.0):
    """[rows, width]: a random block of rows repeated, the last rows their own."""
    g = ref.gen(seed)
    t = torch.empty(rows, width, dtype=dtype, device="cuda")
    block = ref.randn(g, min(rows, 4096), width, std=std, dtype=dtype)
    for at in range(0, rows, block.shape[0]):
        n = min(block.shape[0], rows - at)
        t[at:at + n] = block[:n]
    t[-300:] = ref.randn(g, 300, width, std=std, dtype=dtype)
    return t


def test_products():
    slots, din, dout = 300_001, 7200, 64
    assert slots * din > 1 << 31
    x, w = big(slots, din, BF16, 1), ref.randn(ref.gen(2), 3, dout, din, std=din ** -0.5, dtype=BF16)
    ids = torch.zeros(slots, 1, dtype=torch.int32, device="cuda")
    ids[100_000:], ids[-200:], ids[-50:] = 1, 2, -1
    plan = lm.expert_plan(ids, 3)
    dy = ref.randn(ref.gen(3), slots, dout, dtype=BF16)
    y = lm.expert_product_forward(x, w, plan)
    dx, dw = lm.expert_product_backward(dy, x, w, plan)
    tail = ids[-1000:]
    want = er.product(x[-1000:], w, tail, False, dy[-1000:])
    er.check_product(dict(y=y[-1000:], dx=dx[-1000:], dweight=dw[2:]), {"y": want["y"], "dx": want["dx"], "dweight": tuple(t[2:] for t in want["dweight"])},
                     dict(y=din, dx=dout, dweight=150))
    # the other experts' sums over hundreds of thousands of rows, in parts
    for e, (a, b) in enumerate([(0, 100_000), (100_000, slots - 200)]):
        s, m = (torch.zeros(dout, din, dtype=torch.float64, device="cuda") for _ in range(2))
        for at in range(a, b, 20_000):
            p, q = dy[at:min(b, at + 20_000)].double(), x[at:min(b, at + 20_000)].double()
            s += p.t() @ q
            m += p.abs().t() @ q.abs()
        ref.within(f"dweight {e}", dw[e], s, (b - a + 1) * er.EPS32 * m)


def test_gathered_products():
    tokens, din = 300_001, 7200
    x, w = big(tokens, din, F16, 4), ref.randn(ref.gen(5), 2, 8, din, std=din ** -0.5, dtype=F16)
    ids = (torch.arange(tokens, device="cuda") % 2).int()[:, None]
    plan = lm.expert_plan(ids, 2)
    y = lm.expert_product_forward(x, w, plan, gather=True)
    out = lm.expert_combine_forward(y, None, plan)
    want = er.product(x[-500:], w, ids[-500:], True)["y"]
    at = lm.expert_plan(ids[-500:], 2).places[:, 0].long()
    ref.within("y", out[-500:], want[0][at], (din + 1) * er.EPS32 * want[1][at])


def test_gathered_products_backward():
    """The sorted rows' gradients (fp32) and the tokens are more than 2^31 elements each."""
    tokens, k, din, dout = 300_001, 2, 7200, 64
    x, w = big(tokens, din, BF16, 12), ref.randn(ref.gen(13), 3, dout, din, std=din ** -0.5, dtype=BF16)
    ids = torch.stack([torch.arange(tokens, device="cuda") % 2, torch.arange(tokens, device="cuda") // 150_000 + 1], 1).int()       # (0 or 1, then 1, 2 or none)
    plan = lm.expert_plan(ids, 3)
    dy = ref.randn(ref.gen(14), tokens * k, dout, dtype=BF16)
    dx, dw = lm.expert_product_backward(dy, x, w, plan, gather=True)
    g = dy[plan.places.long()]                                # [tokens, k, dout]
    there = (ids < 3).double()
    for rows in (slice(0, 300), slice(tokens - 600, tokens)):
        s, m = (torch.zeros(x[rows].shape, dtype=torch.float64, device="cuda") for _ in range(2))
        for j in range(k):
            for e in range(3):
                p = g[rows, j].double() * (ids[rows, j] == e).double()[:, None]
                s += p @ w[e].double()
                m += p.abs() @ w[e].double().abs()
        ref.within("dx", dx[rows], s, (dout + k + 1) * er.EPS32 * m)
    for e in range(3):
        s, m = (torch.zeros(dout, din, dtype=torch.float64, device="cuda") for _ in range(2))
        for at in range(0, tokens, 20_000):
            part = x[at:at + 20_000].double()
            for j in range(k):
                p = (g[at:at + 20_000, j].double() * (ids[at:at + 20_000, j] == e).double()[:, None]).t().contiguous()
                s += p @ part
                m += p.abs() @ part.abs()
        ref.within(f"dweight {e}", dw[e], s, (int((ids == e).sum()) + 1) * er.EPS32 * m)
    assert 0 < int(there.sum()) < tokens * k


def test_combination():
    n, k, dim = 150_001, 2, 7200
    assert n * k * dim > 1 << 31
    y, do = big(n * k, dim, BF16, 6), ref.randn(ref.gen(7), n, dim, dtype=BF16)
    ids = torch.randint(0, 4, (n, k), device="cuda", generator=ref.gen(8), dtype=torch.int32)
    ids[-7:] = -1
    plan = lm.expert_plan(ids, 4)
    w = torch.rand(n, k, device="cuda", generator=ref.gen(9))
    out = lm.expert_combine_forward(y, w, plan)
    dy, dw = lm.expert_combine_backward(do, y, w, plan)
    places = plan.places.long()
    rows = slice(n - 600, n - 7)
    terms = w[rows, :, None].double() * y[places[rows]].double()
    ref.within("out", out[rows], terms.sum(1), (k + 1) * er.EPS32 * terms.abs().sum(1))
    ref.within("dy", dy[places[rows]], w[rows, :, None].double() * do[rows, None].double(), er.EPS32 * (w[rows, :, None].double() * do[rows, None].double()).abs())
    prod = y[places[rows]].double() * do[rows, None].double()
    ref.within("dweights", dw[rows], prod.sum(-1), (dim + 1) * er.EPS32 * prod.abs().sum(-1))
    assert not bool(out[-7:].any()) and not bool(dy[-14:].any()) and not bool(dw[-7:].any())


def test_routing_and_plan():
    n, experts, k = (1 << 25) + 5, 70, 2
    assert n * experts > 1 << 31
    z = big(n, experts, F16, 10, std=2.0)
    w, ids, load = lm.route_forward(z, k)
    few = lm.route_forward(z[-1000:], k)
    assert torch.equal(w[-1000:], few[0]) and torch.equal(ids[-1000:], few[1])
    dw = torch.ones_like(w)
    dw[:, 1] = -1.0
    dz = lm.route_backward(dw, load * 1e-7, z, w, ids)
    assert torch.equal(dz[-1000:], lm.route_backward(dw[-1000:], load * 1e-7, z[-1000:], few[0], few[1]))
    total = torch.zeros(experts, dtype=torch.float64, device="cuda")
    for at in range(0, n, 1 << 20):
        total += torch.softmax(z[at:at + (1 << 20)].double(), -1).sum(0)
    # a thread adds 2^13 rows in fp32, then 2^12 of those sums: 2^-24 each of the whole at most
    assert float(((load.double() - total) / total).abs().max()) <= (2 ** 13 + 2 ** 12) * er.EPS32 + ref.F32
    plan = lm.expert_plan(ids, experts)
    rows = torch.sort(ids.view(-1), stable=True)[1]
    assert torch.equal(plan.rows.long(), rows) and int(plan.offsets[-1]) == n * k
    assert torch.equal(plan.places.view(-1)[plan.rows.long()].long(), torch.arange(n * k, device="cuda"))


def test_clipping():
    n = (1 << 31) + 12345
    g = torch.full((n,), 2.0 ** -10, dtype=BF16, device="cuda")
    g[-5:] = 3.0
    small = torch.full((77,), 1.0, device="cuda")
    norm = lm.clip_grads([g, small], 2.0)
    want = ((n - 5) * 2.0 ** -20 + 45.0 + 77.0) ** 0.5
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    c = 2.0 / (want + 1e-6)
    for got, value, u in ((g[0], 2.0 ** -10, BF16), (g[-6], 2.0 ** -10, BF16), (g[-1], 3.0, BF16), (small[-1], 1.0, torch.float32)):
        assert abs(float(got) - value * c) <= value * c * (ref.U[u] + 2.0 ** -22)
    assert bool((g[:-5] == g[0]).all())


def test_wide_rows_of_narrow_results():
    """131072 slots of 2^20 columns: what is counted against the limits is what a pass writes.  Whole numbers, whose sums fp32 holds
    exactly, so that each result is the exact sum rounded once."""
    tokens, k, experts, din, dout = 2048, 64, 3, 1 << 20, 8
    g = ref.gen(11)
    few = lambda *shape: torch.randint(-1, 2, shape, device="cuda", generator=g, dtype=torch.int8).to(BF16)  # noqa: E731
    x, w, dy = few(tokens, din), few(experts, dout, din), few(tokens * k, dout)
    ids = torch.randint(0, experts, (tokens, k), device="cuda", generator=g, dtype=torch.int32)
    plan = lm.expert_plan(ids, experts)
    y = lm.expert_product_forward(x, w, plan, gather=True)
    dx, dw = lm.expert_product_backward(dy, x, w, plan, gather=True, inputs=False)
    assert dx is None
    owner, token = ids.view(-1)[plan.rows.long()].long(), plan.rows.long() // k
    # each token's gradient of each expert, and each token through each expert
    sums = torch.zeros(experts, tokens, dout, dtype=torch.float64, device="cuda")
    sums.index_put_((owner, token), dy.double(), accumulate=True)
    through = torch.zeros(experts, tokens, dout, dtype=torch.float64, device="cuda")
    for at in range(0, din, 1 << 16):
        part = x[:, at:at + (1 << 16)].double()
        for e in range(experts):
            through[e] += part @ w[e, :, at:at + (1 << 16)].double().t().contiguous()
            want = sums[e].t().contiguous() @ part
            assert float(want.abs().max()) < 1 << 24
            assert torch.equal(dw[e, :, at:at + (1 << 16)], want.to(BF16)), (e, at)
    assert float(through.abs().max()) < 1 << 24
    assert torch.equal(y, through[owner, token].to(BF16))
