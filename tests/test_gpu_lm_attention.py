"""Windowed attention with sinks, forward and backward, against 64 bits: types, shared key heads, head widths, one
position to several tiles, windows and sinks around the tiles' borders, masked keys (whatever they hold), rows that
see nothing, strides; splits of the keys; the same bits on every call.

Tolerances (``lm_reference.attention_with_bounds``): every softmax weight and every score gradient is rounded once
to the tensors' type before a product, delta is formed from the rounded output, all else is fp32."""
import pytest
import torch

import lm_reference as ref
import stquant_lm as lm

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def inputs(seed, b, h, hk, t, s, d, dtype):
    g = ref.gen(seed)
    q = ref.randn(g, b, t, h, d, dtype=dtype).transpose(1, 2)
    k, v = (ref.randn(g, b, s, hk, d, dtype=dtype).transpose(1, 2) for _ in range(2))
    return q, k, v, ref.randn(g, b, t, h, d, dtype=dtype).transpose(1, 2)


def check(q, k, v, do, clean=None, **kw):
    """Against the reference on ``clean`` (k, v) where k and v hold what must not matter."""
    out, lse = lm.attention_forward(q, k, v, **kw)
    dq, dk, dv = lm.attention_backward(do, q, k, v, out, lse, **kw)
    kk, vv = clean or (k, v)
    want = ref.attention_with_bounds(q, kk, vv, do, **kw)
    ref.within("out", out, *want["out"])
    wl = want["lse"][0]
    seen = wl > ref.NEG
    assert torch.equal(lse == ref.NEG, ~seen)
    assert float(((lse.double() - wl).abs() - 2.0 ** -17 * (1 + wl.abs()))[seen].max().item() if seen.any() else -1) <= 0
    for name, got in (("dq", dq), ("dk", dk), ("dv", dv)):
        ref.within(name, got, *want[name])
    return out, lse, dq, dk, dv


@pytest.mark.parametrize("t,s", [(1, 1), (1, 65), (2, 2), (31, 31), (33, 100), (64, 64), (65, 65), (128, 128), (129, 200), (300, 300), (3, 1000)])
@pytest.mark.parametrize("d,dtype", [(64, BF16), (128, F16), (8, F16), (72, BF16), (40, BF16), (96, F16)])
def test_causal(t, s, d, dtype):
    check(*inputs(t + s + d, 2, 3, 3, t, s, d, dtype))


@pytest.mark.parametrize("h,hk", [(4, 1), (6, 2), (7, 1), (40, 1), (2, 2)])
@pytest.mark.parametrize("t,s", [(1, 130), (5, 70), (77, 77), (190, 260)])
def test_shared_key_heads(h, hk, t, s):
    check(*inputs(h + t, 2, h, hk, t, s, 64, BF16), window=50, sinks=3)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 0), (63, 0), (64, 1), (65, 64), (100, 65), (128, 200), (1, 130), (400, 5), (0, 7), (1000, 0)])
@pytest.mark.parametrize("t,s", [(330, 330), (90, 390), (1, 390)])
def test_windows_and_sinks(window, sinks, t, s):
    check(*inputs(window + s, 1, 4, 2, t, s, 64, BF16), window=window, sinks=sinks)


@pytest.mark.parametrize("d", [64, 128])
def test_a_window_far_behind_the_first_keys(d):
    """Workgroups whose tiles are the sinks' and then the window's, with many tiles between."""
    check(*inputs(d, 1, 2, 1, 1500, 1500, d, F16), window=130, sinks=70)


@pytest.mark.parametrize("poison", [0.0, float("nan"), float("inf")])
@pytest.mark.parametrize("kind", ["left", "right", "holes", "all", "one"])
def test_masked_keys(kind, poison):
    b, t = 3, 150
    q, k, v, do = inputs(11, b, 4, 2, t, t, 64, BF16)
    mask = torch.ones(b, t, dtype=torch.bool, device="cuda")
    if kind == "left":
        mask[1, :70], mask[2, :149] = False, False
    elif kind == "right":
        mask[1, 70:], mask[2, 1:] = False, False
    elif kind == "holes":
        mask = torch.rand(b, t, device="cuda", generator=ref.gen(1)) < 0.5
    elif kind == "all":
        mask[1:] = False
    else:
        mask[:] = False
        mask[0, 3], mask[1, 149] = True, True
    clean = (k, v)
    if poison != 0.0:
        hide = ~mask[:, None, :, None]
        k, v = k.masked_fill(hide, poison), v.masked_fill(hide, poison)
    for m in (mask, mask.to(torch.uint8)):
        out, lse, dq, dk, dv = check(q, k, v, do, clean, key_mask=m, window=90, sinks=2)
    empty = ~ref.visible(t, t, 90, 2, mask, b, "cuda").any(-1)
    assert not bool(out.transpose(1, 2)[empty].any()) and not bool(dq.transpose(1, 2)[empty].any())
    assert not bool(dk.transpose(1, 2)[~mask].any()) and not bool(dv.transpose(1, 2)[~mask].any())


def test_one_visible_key_has_no_score_gradient():
    """A softmax of one weight is constant: dq and dk are exactly zero."""
    q, k, v, do = inputs(2, 2, 4, 2, 200, 200, 64, BF16)
    out, lse, dq, dk, dv = check(q, k, v, do, window=1)
    assert not bool(dq.any()) and not bool(dk.any())
    mask = torch.zeros(2, 200, dtype=torch.bool, device="cuda")
    mask[:, 5] = True
    _, _, dq, dk, _ = check(q, k, v, do, key_mask=mask)
    assert not bool(dq.any()) and not bool(dk.any())


def test_scores_of_any_size():
    """Scores of +-600: the running maximum carries them, and weights of zero stay zero."""
    q, k, v, do = inputs(3, 1, 2, 2, 200, 200, 64, BF16)
    out, lse = lm.attention_forward(q, k, v, scale=9.0)
    o, wl, p = ref.attention(q, k, v, scale=9.0)
    # the scores' own fp32 error (2^-22 of the products' magnitudes, about 9 * 64) moves every weight alike
    e = 9.0 * (q.double().abs() @ k.double().abs().transpose(-1, -2).contiguous()).max() * 2.0 ** -22
    ref.within("out", out, o, (ref.U[BF16] + ref.F32 + 2 * e) * (p @ v.double().abs()))
    check(q, k, v * 0, do, scale=0.01)


def test_positions_after_a_nan_key_see_it_and_other_batches_do_not():
    q, k, v, _ = inputs(4, 2, 2, 1, 300, 300, 64, F16)
    k = k.clone()
    k[0, 0, 200] = float("nan")
    out, lse = lm.attention_forward(q, k, v)
    assert bool(out[0, :, 200:].isnan().all()) and not bool(out[0, :, :200].isnan().any()) and not bool(out[1].isnan().any())


def test_joint_projection_views_and_gradients_into_one_buffer():
    b, t, h, hk, d = 2, 100, 4, 2, 64
    g = ref.gen(5)
    qkv = ref.randn(g, b, t, (h + 2 * hk) * d, dtype=BF16)
    q, k, v = (x.view(b, t, -1, d).transpose(1, 2) for x in qkv.split([h * d, hk * d, hk * d], -1))
    do = ref.randn(g, b, t, h, d, dtype=BF16).transpose(1, 2)
    want = check(q, k, v, do, window=33, sinks=2)
    buf = torch.zeros_like(qkv)
    grads = tuple(x.view(b, t, -1, d).transpose(1, 2) for x in buf.split([h * d, hk * d, hk * d], -1))
    lm.attention_backward(do, q, k, v, want[0], want[1], window=33, sinks=2, grads=grads)
    assert all(torch.equal(a, w) for a, w in zip(grads, want[2:]))


def test_orders_and_alignments():
    """Head-major, position-major, elements apart, rows off 16 bytes, broadcast heads and gradients: the same values."""
    q, k, v, do = inputs(6, 2, 4, 2, 70, 90, 48, BF16)
    out, lse, dq, dk, dv = check(q, k, v, do)
    flip = lambda x: x.transpose(2, 3).contiguous().transpose(2, 3)  # noqa: E731

    def off(x):
        buf = torch.zeros(x.numel() + 3, dtype=x.dtype, device="cuda")
        y = buf[3:].view(x.shape)
        return y.copy_(x)

    for f in (torch.Tensor.contiguous, flip, off):
        o2, l2 = lm.attention_forward(f(q), f(k), f(v))
        assert torch.equal(o2, out) and torch.equal(l2, lse)
        assert all(torch.equal(a, w) for a, w in zip(lm.attention_backward(f(do), f(q), f(k), f(v), f(out), lse), (dq, dk, dv)))
    ones = torch.ones(1, 1, 1, 1, dtype=BF16, device="cuda").expand(q.shape)
    a = lm.attention_backward(ones, q, k, v, out, lse)
    assert all(torch.equal(x, y) for x, y in zip(a, lm.attention_backward(ones.contiguous(), q, k, v, out, lse)))
    kb = k[:, :1].expand(2, 2, 90, 48)
    assert torch.equal(lm.attention_forward(q, kb, v)[0], lm.attention_forward(q, kb.contiguous(), v)[0])


def test_empty_calls():
    q, k, v, _ = inputs(7, 2, 4, 2, 5, 9, 64, BF16)
    out, lse = lm.attention_forward(q[:, :, :0], k, v)
    assert out.shape == (2, 4, 0, 64) and lse.shape == (2, 4, 0)
    dq, dk, dv = lm.attention_backward(out, q[:, :, :0], k, v, out, lse)
    assert dq.shape == out.shape and not bool(dk.any()) and not bool(dv.any())
    assert lm.attention_forward(q[:0], k[:0], v[:0])[0].shape == (0, 4, 5, 64)


@pytest.mark.parametrize("b,h,hk,t,s,d", [(1, 8, 2, 1, 5000, 128), (1, 3, 1, 30, 3000, 64), (2, 2, 2, 100, 4100, 64)])
def test_split_keys(b, h, hk, t, s, d):
    """Few rows over many keys."""
    q, k, v, do = inputs(s, b, h, hk, t, s, d, BF16)
    check(q, k, v, do)
    mask = torch.ones(b, s, dtype=torch.bool, device="cuda")
    mask[:, 64:2500] = False
    check(q, k, v, do, key_mask=mask)
    check(q, k, v, do, window=700, sinks=130)


@pytest.mark.parametrize("b,h,hk,t,s,d,dtype", [(1, 7, 1, 1100, 1100, 64, BF16), (1, 2, 2, 700, 1500, 128, F16), (2, 40, 2, 70, 600, 72, BF16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 0), (150, 130), (40, 3)])
def test_gradients_of_few_blocks_of_keys(b, h, hk, t, s, d, dtype, window, sinks):
    """Walks in shares, some of them without a row; a batch with masked keys."""
    mask = torch.rand(b, s, device="cuda", generator=ref.gen(s)) < 0.8
    check(*inputs(t + window, b, h, hk, t, s, d, dtype), window=window, sinks=sinks, key_mask=mask)


@pytest.mark.parametrize("d,group,window,sinks", [(64, 1, 64, 3), (128, 1, 100, 200), (64, 3, 1, 1), (128, 2, 300, 128)])
def test_gradients_of_sinks_seen_from_far(d, group, window, sinks):
    """Many blocks of keys: the positions that see the sinks alone are workgroups of their own."""
    mask = torch.ones(4, 1600, dtype=torch.bool, device="cuda")
    mask[1, :2], mask[2, 1:900] = False, False
    check(*inputs(d + window, 4, 8 * group, 8, 1600, 1600, d, BF16), window=window, sinks=sinks, key_mask=mask)


def test_autograd_and_differences():
    q, k, v, do = inputs(8, 2, 4, 2, 60, 60, 64, BF16)
    leaf = [x.clone().requires_grad_(True) for x in (q, k, v)]
    mask = torch.ones(2, 60, dtype=torch.bool, device="cuda")
    mask[1, :20] = False
    kw = dict(window=17, sinks=2, key_mask=mask)
    (lm.attention(*leaf, **kw) * do).sum().backward()
    want = ref.attention_with_bounds(q, k, v, do, **kw)
    g = ref.gen(1)
    for i, name in enumerate(("dq", "dk", "dv")):
        ref.within(name, leaf[i].grad, *want[name])
        d = ref.randn(g, *leaf[i].shape).double()
        num = ref.differences(lambda *a: (ref.attention(*a, **kw)[0] * do.double()).sum(), [q, k, v], i, d, 1e-5)
        allowed = ((want[name][1] + ref.U[BF16] * want[name][0].abs()) * d.abs()).sum() + 1e-5
        assert abs(float(num) - float((leaf[i].grad.double() * d).sum())) <= float(allowed), name


def test_the_same_bits_every_time_on_any_stream_and_in_a_graph():
    q, k, v, do = inputs(9, 2, 6, 2, 260, 260, 64, F16)
    kw = dict(window=100, sinks=5)
    first = check(q, k, v, do, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = lm.attention_forward(q, k, v, **kw)
        again = (out, lse, *lm.attention_backward(do, q, k, v, out, lse, **kw))
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, lse = lm.attention_forward(q, k, v, **kw)
            grads = lm.attention_backward(do, q, k, v, out, lse, **kw)
    for step in range(3):
        q.mul_(0.9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        o2, l2 = lm.attention_forward(q, k, v, **kw)
        assert torch.equal(out, o2) and all(torch.equal(a, b) for a, b in zip(grads, lm.attention_backward(do, q, k, v, o2, l2, **kw))), step


@pytest.mark.parametrize("t,s,window,sinks,masked", [(3, 3, 0, 0, False), (16, 16, 0, 0, False), (17, 17, 0, 0, False), (200, 200, 9, 4, False),
                                                     (200, 200, 16, 1, False), (300, 300, 0, 0, True), (300, 300, 150, 3, True)])
@pytest.mark.parametrize("h,hk,d,dtype", [(4, 2, 64, BF16), (3, 1, 128, F16), (5, 5, 24, BF16)])
def test_rows_of_few_keys_need_no_exact_output(t, s, window, sinks, masked, h, hk, d, dtype):
    """A row of up to 16 keys takes delta from its weights: its dq is the same bits whatever ``out`` holds, and the
    other rows' delta follows ``out``."""
    q, k, v, do = inputs(t + d, 2, h, hk, t, s, d, dtype)
    mask = None
    if masked:
        mask = torch.rand(2, s, device="cuda", generator=ref.gen(t)) < 0.5
        mask[1, :260] = False
    kw = dict(window=window, sinks=sinks, key_mask=mask)
    out, lse, dq, _, _ = check(q, k, v, do, **kw)
    other, _, _ = lm.attention_backward(do, q, k, v, out + 1, lse, **kw)
    count = ref.visible(t, s, window, sinks, mask, 2, "cuda").sum(-1)
    few = count <= 16
    same = (dq == other).all(-1).transpose(1, 2)              # [batch, position, head]
    assert bool(same[few].all())
    if bool((~few).any()):
        assert not bool(same[~few].all())
