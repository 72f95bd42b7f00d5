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
