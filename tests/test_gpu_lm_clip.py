"""The global gradient norm and clipping against 64 bits: mixed types, ragged lists of any length, unaligned views, values
whose squares are no floats, in place and apart.

Tolerances: the norm is rounded once to fp32 (squares and sums are 64 bits), the scale once, and the scaled gradient
once in fp32 and once to its type."""
import pytest
import torch

import lm_expert_reference as er
import lm_reference as ref
import stquant_lm as lm

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def check(grads, max_norm, out=None):
    before = [g.clone() for g in grads]
    norm = lm.clip_grads(grads, max_norm, out=out)
    want, scaled = er.clip(before, max_norm)
    assert norm.dtype == F32 and norm.shape == ()
    # (64-bit sums in another order: 2^-40 covers 2^12 roundings each way)
    assert abs(float(norm) - want) <= want * (2.0 ** -24 + 2.0 ** -40), (float(norm), want)
    for i, (g, b, o, s) in enumerate(zip(grads, before, grads if out is None else out, scaled)):
        ref.within(f"gradient {i}", o, s, 2.0 ** -23 * s.abs())
        if out is not None:
            assert torch.equal(g, b)
    assert float(lm.grad_norm(before)) == float(norm)
    return norm


def tensors(sizes, dtype, seed=0, std=1e-2):
    g = ref.gen(seed)
    return [ref.randn(g, n, std=std, dtype=dtype) for n in sizes]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes", [[1], [0, 5, 0], [7, 8, 9, 4095, 4096, 4097], [16383, 16384, 16385, 32769], [1 << 20, 3, (1 << 20) + 5], [3] * 127, [1] * 128,
                                   [17] * 129, [5, 0] * 700, [40000] * 300])
@pytest.mark.parametrize("apart", [False, True])
def test_against_64_bits(sizes, dtype, apart):
    grads = tensors(sizes, dtype)
    norm = float(lm.grad_norm(grads))
    check(grads, 0.3 * norm, out=[torch.full_like(g, 7.0) for g in grads] if apart else None)


@pytest.mark.parametrize("count", [159, 160, 161, 319, 320, 321])
@pytest.mark.parametrize("empty", [None, 0, 159, 160])
@pytest.mark.parametrize("apart", [False, True])
def test_lists_that_end_at_a_launch(count, empty, apart):
    """A launch holds 160 tensors (empty ones take no place): lists around one and two of them, with an empty tensor at the cut."""
    sizes = [1 + 37 * i % 101 for i in range(count)]
    if empty is not None and empty < count:
        sizes[empty] = 0
    grads = [t for i, n in enumerate(sizes) for t in tensors([n], (F32, BF16, F16)[i % 3], seed=i)]
    check(grads, 0.05, out=[torch.full_like(g, 7.0) for g in grads] if apart else None)


def test_mixed_types():
    grads = [t for d in (F32, BF16, F16) for t in tensors([1000, 33, 70000], d, seed=3)]
    check(grads, 0.1)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_views_that_start_anywhere(dtype):
    flat, out = tensors([400000], dtype)[0], torch.zeros(400000, dtype=dtype, device="cuda")
    cuts = [0, 1, 4, 11, 12, 20000, 20001, 53333, 200001, 400000]
    views = lambda t: [t[a:b] for a, b in zip(cuts, cuts[1:])]  # noqa: E731
    check(views(flat), 0.5, out=views(out))
    keep = flat.clone()
    inner = [flat[3:70000], flat[70001:70002], flat[80005:399999]]
    check(inner, 0.01)
    hole = torch.ones(400000, dtype=torch.bool, device="cuda")
    hole[3:70000], hole[70001:70002], hole[80005:399999] = False, False, False
    assert torch.equal(flat[hole], keep[hole])                    # nothing beside them is written


def test_shapes_and_orders():
    g = ref.gen(9)
    a = ref.randn(g, 6, 50, 70)
    grads = [a[0], a[1].t(), a[2:4].permute(2, 0, 1), ref.randn(g, 2, 3, 4, 5).to(memory_format=torch.channels_last), torch.tensor(3.0, device="cuda")]
    check(grads, 1.0)
    out = [torch.empty_like(x) for x in grads]
    check(grads, 0.1, out=out)
    with pytest.raises(RuntimeError, match="gradients must be dense"):
        lm.clip_grads([a[:, :3]], 1.0)
    with pytest.raises(RuntimeError, match="out must be like its gradient"):
        lm.clip_grads([a[1].t()], 1.0, out=[torch.empty(70, 50, device="cuda")])


def test_no_clipping_below_the_norm():
    """A scale of 1 leaves the bits alone, and copies them where the result goes elsewhere."""
    grads = tensors([1000, 77], BF16)
    before = [g.clone() for g in grads]
    out = [torch.zeros_like(g) for g in grads]
    lm.clip_grads(grads, 1e6, out=out)
    lm.clip_grads(grads, 1e6)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(grads, before, out))


@pytest.mark.parametrize("dtype,value", [(F32, 3e38), (F32, 1e-38), (F32, 1e-45), (BF16, 3e38), (F16, 65504.0), (F16, 6e-8)])
def test_values_whose_squares_are_no_floats(dtype, value):
    grads = [torch.full((5000,), value, dtype=dtype, device="cuda"), torch.zeros(9, dtype=dtype, device="cuda")]
    exact = float(grads[0][0].double()) * 5000 ** 0.5
    norm = lm.clip_grads(grads, 1.0)
    if exact > 3.4e38:                        # the sum is finite, its float is not: the scale is formed from the sum
        assert float(norm) == float("inf")
        want = float(torch.tensor(value, dtype=dtype).double()) / exact
        assert abs(float(grads[0][0]) - want) <= want * (2 * ref.U[dtype] + 2.0 ** -22)
    else:
        assert abs(float(norm) - exact) <= exact * 2.0 ** -23 + 1e-45


def test_nan_and_infinity():
    for bad in (float("nan"), float("inf"), float("-inf")):
        grads = [torch.ones(100, device="cuda"), torch.ones(3, device="cuda", dtype=BF16)]
        grads[0][7] = bad
        norm = lm.clip_grads(grads, 1.0)
        assert bool(torch.isnan(norm)) == (bad != bad)
        if bad == bad:
            assert float(norm) == float("inf") and bool(torch.isnan(grads[0][7])) and float(grads[0].nan_to_num().abs().max()) == 0.0 and not bool(grads[1].any())
        else:
            assert bool(torch.isnan(grads[0]).all()) and bool(torch.isnan(grads[1]).all())


def test_an_infinite_limit():
    """It leaves the bits alone, and of an infinite norm makes inf / inf."""
    g = tensors([500, 33], BF16)
    before = [t.clone() for t in g]
    assert float(lm.clip_grads(g, float("inf"))) == float(lm.grad_norm(before)) and all(torch.equal(a, b) for a, b in zip(g, before))
    g[0][3] = float("inf")
    assert float(lm.clip_grads(g, float("inf"))) == float("inf") and bool(torch.isnan(g[0]).all()) and bool(torch.isnan(g[1]).all())


def test_zero_norms_and_limits():
    z = [torch.zeros(500, device="cuda")]
    assert float(lm.clip_grads(z, 1.0)) == 0.0 and not bool(z[0].any())
    g = tensors([500], F32)
    lm.clip_grads(g, 0.0)
    assert not bool(g[0].any())
    e = [torch.zeros(0, device="cuda")]
    assert float(lm.clip_grads(e, 1.0)) == 0.0 and float(lm.grad_norm(e)) == 0.0


def test_a_given_norm():
    """Ranks add the squares of their norms and scale by the root."""
    shards = [tensors([3000, 11], F32, seed=s) for s in (1, 2)]
    norm = sum(lm.grad_norm(s).double() ** 2 for s in shards).sqrt().float()
    whole = [g.clone() for s in shards for g in s]
    want, scaled = er.clip(whole, 0.2, float(norm))
    for s in shards:
        assert lm.clip_grads(s, 0.2, norm=norm) is norm
    for got, w in zip([g for s in shards for g in s], scaled):
        ref.within("gradient", got, w, 2.0 ** -22 * w.abs())
    with pytest.raises(RuntimeError, match="norm must be one float32"):
        lm.clip_grads(whole, 1.0, norm=norm.double())


def test_against_torch():
    ps = [torch.nn.Parameter(t) for t in tensors([300, 4000, 77], F32)]
    for p, g in zip(ps, tensors([300, 4000, 77], F32, seed=1, std=1.0)):
        p.grad = g.clone()
    mine = [p.grad.clone() for p in ps]
    a, b = lm.clip_grads(mine, 2.0), torch.nn.utils.clip_grad_norm_(ps, 2.0)
    assert abs(float(a) - float(b)) <= 1e-5 * float(b)
    for x, p in zip(mine, ps):
        assert float((x - p.grad).abs().max()) <= 1e-5 * float(p.grad.abs().max())


def test_clipped_gradients_count_as_changed():
    x = torch.ones(10, device="cuda", requires_grad=True)
    g = torch.ones(10, device="cuda") * 5
    y = (x * g).sum()                          # saves g
    lm.clip_grads([g], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_overlapping_gradients_are_refused():
    t = torch.ones(100, device="cuda")
    for grads in ([t, t], [t[:60], t[50:]], [t, t[3:4]]):
        with pytest.raises(RuntimeError, match="must not overlap"):
            lm.clip_grads(grads, 1.0)
    assert abs(float(lm.grad_norm([t, t])) - 200 ** 0.5) <= 1e-5
