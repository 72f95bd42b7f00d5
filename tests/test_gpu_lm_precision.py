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
