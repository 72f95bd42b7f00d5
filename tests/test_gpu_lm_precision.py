"""Where 16 bits of the attention's score gradients and weights could run out: fp16's small numbers, rows in which one
weight is nearly all, scores of hundreds; against 64 bits."""
import pytest
import torch

import lm_reference as ref
import stquant_lm as lm

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def rms(x):
    return float(x.double().square().mean().sqrt())


def near(name, got, want, steps):
    """Root mean squares: the error is that of rounding ``want`` once (a tenth more), and ``steps`` relative roundings of
    the terms on the way, each as if all of them went the same way."""
    once = rms(want.to(got.dtype).double() - want)
    off, most = rms(got.double() - want), 1.1 * once + steps * ref.U[got.dtype] * rms(want)
    print(f"{name}: off {off / rms(want):.2e} of the values, rounded once {once / rms(want):.2e}, allowed {most / rms(want):.2e}", flush=True)
    assert off <= most, name


@pytest.mark.parametrize("std", [1e-4, 1e-3, 1e-2, 1.0, 300.0])
@pytest.mark.parametrize("h,hk,t,s,d,window", [(2, 1, 500, 4500, 64, 0), (1, 1, 3100, 3100, 128, 2500)])
def test_fp16_score_gradients_keep_their_bits(std, h, hk, t, s, d, window):
    """Score gradients of rows with thousands of keys are about |dout| / keys: below 2^-14 fp16 holds fewer bits of them.

    Two roundings of the terms (the score gradients', and delta's from the rounded output)."""
    g = ref.gen(t + d)
    q = ref.randn(g, 1, h, t, d, dtype=F16)
    k, v = (ref.randn(g, 1, hk, s, d, dtype=F16) for _ in range(2))
    do = ref.randn(g, 1, h, t, d, std=std, dtype=F16)
    out, lse = lm.attention_forward(q, k, v, window=window)
    got = lm.attention_backward(do, q, k, v, out, lse, window=window)
    want = ref.attention_with_bounds(q, k, v, do, window=window)
    for name, x in zip(("dq", "dk", "dv"), got):
        near(name, x, want[name][0], 2)


@pytest.mark.parametrize("gap", [17, 18, 19])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("keys", [2, 5, 16])
@pytest.mark.parametrize("scale", [1.0, 40.0])
def test_a_nearly_certain_row_keeps_all_its_score_gradients(gap, dtype, keys, scale):
    """One weight of 1 - 2^-gap, the rest on another key: both keys' score gradients are alike in size, and dq is their
    difference times that of the keys.

    The score gradients go into the products as two parts (2^-16 of them is left); around them stands fp32's error of the
    products with dout (64 roundings of 2^-24, at random 2^-21 of the magnitudes; twice that), and of the weights, 2^-21
    (3 + |lse|) of each, alike for a row's keys."""
    d, rows = 64, 8
    q, k, v = (torch.zeros(1, rows, n, d, device="cuda") for n in (1, keys, keys))
    q[..., 0] = 4.0
    k[..., 0] = -30.0 / scale                    # keys that weigh nothing: 2^-43 and less
    k[:, :, 0, 0], k[:, :, -1, 0] = 2.0, 2.0 - gap * 0.6931471805599453 / (4.0 * scale)
    g = ref.gen(gap + keys)
    k[:, :, 0, 1:], k[:, :, -1, 1:] = ref.randn(g, 1, rows, d - 1), ref.randn(g, 1, rows, d - 1)
    v[:, :, 0], v[:, :, -1] = ref.randn(g, 1, rows, d), ref.randn(g, 1, rows, d, std=32.0)
    do = ref.randn(g, 1, rows, 1, d, dtype=dtype)
    q, k, v = (x.to(dtype) for x in (q, k, v))
    out, lse = lm.attention_forward(q, k, v, scale=scale)
    got = lm.attention_backward(do, q, k, v, out, lse, scale=scale)
    o, wl, p = ref.attention(q, k, v, scale=scale)
    dp = do.double() @ v.double().transpose(-1, -2).contiguous()
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    mag = do.double().abs() @ v.double().abs().transpose(-1, -2).contiguous()
    e = p * scale * 2.0 ** -20 * (mag + (p * mag).sum(-1, keepdim=True)) + ds.abs() * (2.0 ** -16 + 2.0 ** -21 * (3 + wl.abs()[..., None]))
    assert float((p[..., 0].amin())) > 1 - 2.0 ** -16 and float(p[..., 0].amax()) < 1 - 2.0 ** -20
    ref.within("dq", got[0], ds @ k.double(), e @ k.double().abs())
    ref.within("dk", got[1], ds.transpose(-1, -2).contiguous() @ q.double(), e.transpose(-1, -2).contiguous() @ q.double().abs())


def test_a_row_of_one_key_has_no_score_gradient_at_any_score():
    """Exactly zero, whatever the size of the score, and in rows beside ones that see more."""
    for scale in (1e-3, 1.0, 9.0, 300.0):
        for dtype in (BF16, F16):
            g = ref.gen(5)
            q, k, v, do = (ref.randn(g, 2, 3, 90, 64, dtype=dtype) for _ in range(4))
            out, lse = lm.attention_forward(q, k, v, scale=scale)
            dq, dk, dv = lm.attention_backward(do, q, k, v, out, lse, scale=scale)
            assert not bool(dq[:, :, 0].any()) and bool(dq[:, :, 1:].any())
            mask = torch.zeros(2, 90, dtype=torch.bool, device="cuda")
            mask[0, 7], mask[1, 70] = True, True
            out, lse = lm.attention_forward(q, k, v, scale=scale, key_mask=mask)
            dq, dk, dv = lm.attention_backward(do, q, k, v, out, lse, scale=scale, key_mask=mask)
            assert not bool(dq.any()) and not bool(dk.any()) and bool(dv.any())


@pytest.mark.parametrize("t,s,window", [(200, 200, 0), (70, 300, 90)])
@pytest.mark.parametrize("h,hk,d,dtype", [(2, 2, 64, BF16), (4, 2, 128, F16)])
@pytest.mark.parametrize("scale", [3.0, 9.0])
def test_gradients_of_scores_in_the_hundreds(t, s, window, h, hk, d, dtype, scale):
    """Peaked rows, |lse| of hundreds: the weights carry fp32's error of the scores and of lse, 2^-22 of their magnitudes."""
    g = ref.gen(t + d)
    q, do = (ref.randn(g, 1, h, t, d, dtype=dtype) for _ in range(2))
    k, v = (ref.randn(g, 1, hk, s, d, dtype=dtype) for _ in range(2))
    kw = dict(window=window, scale=scale)
    out, lse = lm.attention_forward(q, k, v, **kw)
    got = lm.attention_backward(do, q, k, v, out, lse, **kw)
    want = ref.attention_with_bounds(q, k, v, do, **kw)
    e = 2.0 ** -22 * scale * float((q.double().abs() @ k.double().abs().repeat_interleave(h // hk, 1).transpose(-1, -2).contiguous()).max())
    _, wl, p = ref.attention(q, k, v, **kw)
    assert float(wl.abs().max()) > 60 and float(p.amax(-1).median()) > 0.9
    kk, vv = (x.double().repeat_interleave(h // hk, 1) for x in (k, v))
    dp = do.double() @ vv.transpose(-1, -2).contiguous()
    # (weights below fp32's and bfloat16's smallest normal number are 0, and score gradients too)
    see = ref.visible(t, s, window, 0, None, 1, "cuda")[:, None]
    eds = 2 * e * p * scale * (dp.abs() + (p * dp.abs()).sum(-1, keepdim=True)) + see * 2.0 ** -125 * scale * (1 + dp.abs() + dp.abs().amax(-1, keepdim=True))
    tr = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    shared = lambda x: x.reshape(1, hk, h // hk, s, d).sum(2)  # noqa: E731
    more = {"dq": eds @ kk.abs(), "dk": shared(tr(eds) @ q.double().abs()), "dv": shared(tr(2 * e * p + see * 2.0 ** -125) @ do.double().abs())}
    assert bool(got[0].any()) and bool(got[1].any())
    for name, x in zip(("dq", "dk", "dv"), got):
        ref.within(name, x, want[name][0], want[name][1] + more[name])


@pytest.mark.parametrize("d", [64, 128])
def test_fp16_weights_of_long_contexts_keep_their_bits(d):
    """Normalised weights over 200,000 keys are 2^-18 on average, below fp16's full precision (2^-14): one rounding of
    them in dv."""
    g = ref.gen(d)
    q, do = ref.randn(g, 1, 1, 64, d, dtype=F16), ref.randn(g, 1, 1, 64, d, std=100.0, dtype=F16)
    k, v = (ref.randn(g, 1, 1, 200_000, d, dtype=F16) for _ in range(2))
    out, lse = lm.attention_forward(q, k, v)
    dv = lm.attention_backward(do, q, k, v, out, lse)[2]
    _, wl, p = ref.attention(q, k, v)
    near("dv", dv, p.transpose(-1, -2).contiguous() @ do.double(), 1)
    assert float((lse.double() - wl).abs().max()) <= 2.0 ** -17 * (1 + float(wl.abs().max()))


def test_fp16_a_key_far_above_many():
    """A first key 17 above 2^20 others: each of those weighs e^-17, 0.7 of fp16's smallest number, together 4 %.

    The weights' rounding, alike for all of them, and the sum's of 16,384 tiles, 2^-25 of about one each: 2^-11 both."""
    n = 1 << 20
    heads = 256                                   # (so many that one walk takes all keys)
    q, k = torch.zeros(1, 1, 1, 64, dtype=F16, device="cuda"), torch.zeros(1, 1, n, 64, dtype=F16, device="cuda")
    q[..., 0], k[:, :, 0, 0] = 4.0, 4.25
    v = torch.ones(1, 1, n, 64, dtype=F16, device="cuda")
    v[:, :, 0] = 0.0
    k, v = k.expand(1, heads, n, 64), v.expand(1, heads, n, 64)
    for rows in (1, 40):                          # one wave's rows, and a workgroup's
        out, lse = lm.attention_forward(q.expand(1, heads, rows, 64), k, v, scale=1.0)
        own = torch.arange(n - rows, n, device="cuda", dtype=torch.float64)[:, None]
        total = own * torch.exp(torch.tensor(-17.0, dtype=torch.float64))
        want = (total / (1 + total)).expand(rows, 64)
        ref.within("out", out[0], want.expand(heads, rows, 64), 2.0 ** -10 * want)
        assert float((lse[0].double() - (17 + torch.log1p(total[:, 0]))).abs().max()) <= 2.0 ** -11 + 2.0 ** -17 * 17


@pytest.mark.parametrize("d,group,window,sinks", [(64, 1, 64, 3), (128, 1, 100, 200), (64, 3, 1, 1), (128, 2, 300, 128)])
def test_every_far_row_reaches_the_sinks(d, group, window, sinks):
    """dout is zero in all rows of a head but one: what the sinks' keys get is that row's, wherever the walk is cut.

    Rows around every multiple of 32 behind the window, one a head, so that a row lost at any border leaves dv zero."""
    t, hk = 1600, 40
    h = hk * group
    rows = [p + i for p in range(window + sinks + 130, t, 64) for i in (-1, 0, 1)][: 4 * h]
    g = ref.gen(window)
    q = ref.randn(g, 4, h, t, d, std=0.3, dtype=F16)
    k, v = (ref.randn(g, 4, hk, t, d, std=0.3, dtype=F16) for _ in range(2))
    do = torch.zeros_like(q)
    at = [(i // h, i % h, p) for i, p in enumerate(rows)]
    for b, j, p in at:
        do[b, j, p] = ref.randn(g, d, std=30.0, dtype=F16)
    out, lse = lm.attention_forward(q, k, v, window=window, sinks=sinks)
    dv = lm.attention_backward(do, q, k, v, out, lse, window=window, sinks=sinks)[2]
    want = torch.zeros(4, hk, t, d, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(want)
    see = ref.visible(t, t, window, sinks, None, 1, "cuda")[0]
    for b, j, p in at:
        s = (q[b, j, p].double() @ k[b, j // group].double().t().contiguous() * d ** -0.5).masked_fill(~see[p], ref.NEG)
        w = torch.softmax(s, -1)[:, None] * do[b, j, p].double()[None]
        want[b, j // group] += w
        mag[b, j // group] += w.abs()
    assert float(want[:, :, :sinks].abs().amax()) > 0.01
    ref.within("dv", dv, want, (ref.U[F16] + ref.F32) * mag)
