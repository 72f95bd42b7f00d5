"""The operators inside autograd: second derivatives are refused, tensors written in place are known to be."""
import pytest
import torch

import lm_reference as ref
import stquant_lm as lm

pytestmark = pytest.mark.gpu


def calls():
    g = ref.gen(1)
    tok = torch.randint(0, 20, (30,), device="cuda", generator=g)
    f = lambda *s, dtype=torch.float32: ref.randn(g, *s, dtype=dtype).requires_grad_(True)  # noqa: E731
    return {
        "embedding": (lambda w: lm.embedding(tok, w), [f(20, 16)]),
        "norm_residual": (lambda x, b, w: sum(lm.norm_residual(x, b, w)), [f(9, 32), f(9, 32), f(32)]),
        "attention": (lm.attention, [f(1, 2, 20, 16, dtype=torch.bfloat16) for _ in range(3)]),
        "distill_loss": (lambda z: lm.distill_loss(z, torch.zeros(7, 2, device="cuda"), tok[:14].view(7, 2)), [f(7, 40)]),
    }


@pytest.mark.parametrize("name", ["embedding", "norm_residual", "attention", "distill_loss"])
def test_second_derivatives_are_refused(name):
    """The gradients are not differentiable: torch says so, rather than take them for constants."""
    fn, leaves = calls()[name]
    y = fn(*leaves)
    grads = torch.autograd.grad((y * y).sum(), leaves, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        sum(x.float().square().sum() for x in grads).backward()


def test_what_is_written_in_place_counts_as_changed():
    """A tensor that another node saved and an operator then wrote: its backward pass refuses rather than use it."""
    g = ref.gen(2)
    teacher, ids = torch.zeros(6, 3, device="cuda"), torch.randint(0, 50, (6, 3), device="cuda", generator=g)

    def capped():
        z = ref.randn(g, 6, 50).requires_grad_(True)
        return z, torch.tanh(z)                  # (saves its result)

    z, y = capped()
    with torch.no_grad():
        _, dz = lm.distill_loss_and_grad(y.detach(), teacher, ids, grad=1.0, out=y.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dz)
    z, y = capped()
    _, stats = lm.distill_loss_forward(y.detach(), teacher, ids)
    dz = lm.distill_loss_backward(1.0, y.detach(), teacher, ids, stats, out=y.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dz)
    tok = torch.randint(0, 50, (4,), device="cuda", generator=g)
    w = ref.randn(g, 50, 8).requires_grad_(True)
    y = torch.tanh(w)
    lm.embedding_backward(torch.ones(4, 8, device="cuda"), tok, 50, out=y.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    q, k, v = (ref.randn(g, 1, 2, 10, 16, dtype=torch.bfloat16) for _ in range(3))
    out, lse = lm.attention_forward(q, k, v)
    buf = [torch.zeros_like(q) for _ in range(3)]
    before = [b._version for b in buf]
    lm.attention_backward(torch.ones_like(q), q, k, v, out, lse, grads=buf)
    assert all(b._version > n for b, n in zip(buf, before))


def test_in_place_calls_in_inference_mode():
    with torch.inference_mode():
        z, t, ids = torch.zeros(3, 10, device="cuda"), torch.zeros(3, 2, device="cuda"), torch.ones(3, 2, dtype=torch.int64, device="cuda")
        want = lm.distill_loss_and_grad(z, t, ids, grad=1.0)[1]
        assert torch.equal(lm.distill_loss_and_grad(z, t, ids, grad=1.0, out=z)[1], want)
