"""The residual norms, forward and backward, against 64 bits: both kinds, with and without the norm after the
block, gates of every grouping, widths of one wave and of a workgroup, odd widths and strides.

Tolerances: a row's values carry 2^-17 of the row's largest magnitude (fp32 sums and the deviation), times the
operand magnitudes that multiply them, before their one rounding; the column sums the same of the terms' magnitudes."""
import pytest
import torch

import lm_reference as ref
import stquant_lm as lm

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NAMES = ("x", "block", "pre_weight", "pre_bias", "post_weight", "post_bias", "gate")


def operands(seed, n, d, dtype, kind, post, gate, wdt=None):
    g, wdt = ref.gen(seed), wdt or dtype
    layer = kind == "layer"
    vec = lambda on, mean: ref.randn(g, d, std=0.2, mean=mean, dtype=wdt) if on else None  # noqa: E731
    return dict(x=ref.randn(g, n, d, std=1.5, mean=0.5 * layer, dtype=dtype), block=ref.randn(g, n, d, std=0.6, mean=1.0 * layer, dtype=dtype),
                pre_weight=vec(True, 1.0), pre_bias=vec(layer, 0.1), post_weight=vec(post, 1.0), post_bias=vec(layer and post, 0.0),
                gate=ref.randn(g, gate, d, std=0.5, dtype=wdt) if gate else None)


def reference(o, scale, eps, kind, dr, dh):
    leaf = {k: None if o[k] is None else o[k].double().detach().requires_grad_(True) for k in NAMES}
    r, h = ref.norm_residual(*(leaf[k] for k in NAMES), scale, eps, kind)
    have = [k for k in NAMES if o[k] is not None]
    grads = torch.autograd.grad([r, h], [leaf[k] for k in have], [torch.zeros_like(r) if dr is None else dr.double(), dh.double()])
    return r.detach(), h.detach(), dict(zip(have, grads))


def row_bound(want):
    return ref.F32 * 4 * want.abs().amax(-1, keepdim=True)


def check(o, kind, scale=0.8, eps=1e-5, with_dr=True, seed=99):
    x = o["x"]
    g = ref.gen(seed)
    dr, dh = ref.randn(g, *x.shape, dtype=x.dtype) if with_dr else None, ref.randn(g, *x.shape, dtype=x.dtype)
    kw = {k: o[k] for k in NAMES[3:]}
    r, h, stats = lm.norm_residual_forward(x, o["block"], o["pre_weight"], residual_scale=scale, eps=eps, kind=kind, **kw)
    got = lm.norm_residual_backward(dr, dh, x, o["block"], o["pre_weight"], stats, residual_scale=scale, kind=kind, **kw)
    want_r, want_h, want = reference(o, float(torch.tensor(scale)), eps, kind, dr, dh)
    ref.within("r", r, want_r, row_bound(want_r))
    ref.within("h", h, want_h, row_bound(want_h))
    assert set(got) == set(want)
    for k in ("x", "block"):
        ref.within("d" + k, got[k], want[k], 4 * row_bound(want[k]))
    # the column sums: what the terms of the sum measure (normalised values up to 8, output gradients up to 6)
    n = x.numel() // x.shape[-1]
    for k in NAMES[2:]:
        if k in got:
            ref.within("d" + k, got[k], want[k], ref.F32 * 16 * n ** 0.5 * (1 + want[k].abs().max()) * torch.ones_like(want[k]))
    return r, h, stats, got


@pytest.mark.parametrize("n,d", [(1, 8), (3, 9), (5, 768), (130, 100), (64, 1024), (33, 1025), (7, 4096), (20, 4095), (5, 5003), (4, 8192), (2100, 72)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("kind,post,gated", [("rms", False, 0), ("layer", False, 1), ("rms", True, 1), ("layer", True, 0)])
def test_against_64_bits(n, d, dtype, kind, post, gated):
    check(operands(n + d, n, d, dtype, kind, post, gated), kind)


@pytest.mark.parametrize("groups", [1, 2, 60, 600, 1200])
@pytest.mark.parametrize("d", [40, 1160])
def test_gates_of_groups(groups, d):
    """One gate for all rows, for runs of them, and one each (more groups than workgroups)."""
    check(operands(groups, 1200, d, BF16, "rms", True, groups), "rms")


@pytest.mark.parametrize("d", [768, 2048])
def test_fp32_weights_under_16_bit_rows(d):
    _, _, _, got = check(operands(d, 50, d, BF16, "layer", True, 1, wdt=F32), "layer")
    assert got["pre_weight"].dtype == F32 and got["gate"].dtype == F32


def test_without_a_gradient_of_r():
    check(operands(1, 77, 96, F32, "rms", False, 0), "rms", with_dr=False)


@pytest.mark.parametrize("shift,pad", [(0, 8), (1, 0), (0, 3), (4, 4)])
def test_strided_rows(shift, pad):
    n, d = 40, 264
    o = operands(7, n, d, BF16, "layer", True, 1)
    for k in ("x", "block"):
        buf = torch.zeros(n * (d + pad) + shift, dtype=BF16, device="cuda")
        view = buf[shift:].view(n, d + pad)[:, :d]
        view.copy_(o[k])
        o[k] = view
    check(o, "layer")


def test_leading_shapes_and_transposed_rows():
    o = operands(2, 6 * 5, 64, F32, "rms", True, 6)
    r, h, _, got = check(o, "rms")
    kw = {k: o[k] for k in NAMES[3:]}
    kw["gate"] = o["gate"].view(6, 1, 64)
    x3, b3 = o["x"].view(6, 5, 64), o["block"].view(6, 5, 64).transpose(0, 1).contiguous().transpose(0, 1)
    r3, h3, st = lm.norm_residual_forward(x3, b3, o["pre_weight"], residual_scale=0.8, **kw)
    assert r3.shape == (6, 5, 64) and torch.equal(r3.view(-1, 64), r) and torch.equal(h3.view(-1, 64), h)


def test_rows_far_from_zero():
    """A mean 1000 times the deviation: the deviation is taken from the mean, not from a difference of squares."""
    o = operands(3, 16, 512, F32, "layer", True, 0)
    o["block"] = o["block"] * 0.01 + 10.0
    want_r, want_h, _ = reference(o, 1.0, 1e-5, "layer", None, torch.zeros_like(o["x"]))
    r, h, _ = lm.norm_residual_forward(o["x"], o["block"], o["pre_weight"], kind="layer", **{k: o[k] for k in NAMES[3:]})
    # the inputs' own spacing at 10 is 2^-20.7: (y - mean) / 0.006 carries up to 2^-24 * 10 / 0.006 of error from the mean
    ref.within("r", r, want_r, 2.0 ** -24 * 10 / 0.006 * 4 * torch.ones_like(want_r))


def test_zero_rows_and_nan_rows():
    o = operands(4, 6, 128, F32, "rms", True, 0)
    o["x"][2] = 0
    o["block"][2] = 0
    o["block"][4, 3] = float("nan")
    kw = {k: o[k] for k in NAMES[3:]}
    r, h, st = lm.norm_residual_forward(o["x"], o["block"], o["pre_weight"], **kw)
    assert bool((r[2] == 0).all()) and bool((h[2] == 0).all())
    assert bool(r[4].isnan().all()) and not bool(r[[0, 1, 2, 3, 5]].isnan().any()) and not bool(h[[0, 1, 2, 3, 5]].isnan().any())


def test_empty_calls():
    o = operands(5, 0, 64, F32, "rms", True, 1)
    kw = {k: o[k] for k in NAMES[3:]}
    r, h, st = lm.norm_residual_forward(o["x"], o["block"], o["pre_weight"], **kw)
    got = lm.norm_residual_backward(None, h, o["x"], o["block"], o["pre_weight"], st, **kw)
    assert r.shape == h.shape == (0, 64)
    assert all(bool((got[k] == 0).all()) for k in ("pre_weight", "post_weight", "gate"))


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_autograd_and_differences(kind):
    o = operands(6, 24, 56, F32, kind, True, 3)
    leaf = {k: None if o[k] is None else o[k].clone().requires_grad_(True) for k in NAMES}
    g = ref.gen(12)
    ur, uh = ref.randn(g, 24, 56), ref.randn(g, 24, 56)
    r, h = lm.norm_residual(leaf["x"], leaf["block"], leaf["pre_weight"], residual_scale=0.5, eps=1e-6, kind=kind, **{k: leaf[k] for k in NAMES[3:]})
    ((r * ur).sum() + (h * uh).sum()).backward()
    args = [None if o[k] is None else o[k].double() for k in NAMES]

    def f(*a):
        rr, hh = ref.norm_residual(*a, 0.5, 1e-6, kind)
        return (rr * ur.double()).sum() + (hh * uh.double()).sum()

    for i, k in enumerate(NAMES):
        if o[k] is None:
            continue
        d = ref.randn(g, *o[k].shape).double()
        num, ana = float(ref.differences(f, args, i, d, 1e-5)), float((leaf[k].grad.double() * d).sum())
        # the gradient's own tolerance over all its elements, and the differences' 1e-10 of third derivatives
        assert abs(num - ana) <= 16 * ref.F32 * float((leaf[k].grad.double().abs() * d.abs()).sum()) + 1e-6, k
    leaf["x"].grad = None
    lm.norm_residual(leaf["x"], leaf["block"], leaf["pre_weight"], kind=kind, **{k: leaf[k] for k in NAMES[3:]})[0].sum().backward()
    assert torch.equal(leaf["x"].grad, torch.ones_like(o["x"]))


def test_the_same_bits_every_time():
    o = operands(9, 3000, 768, BF16, "layer", True, 1)
    a = check(o, "layer")
    b = check(o, "layer")
    assert all(torch.equal(a[3][k], b[3][k]) for k in a[3])
