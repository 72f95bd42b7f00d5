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
