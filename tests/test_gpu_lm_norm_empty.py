"""Residual norms of no rows."""
import pytest
import torch

import stquant_lm as lm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("groups", [1, 2, 7, 70_000])
def test_gates_of_no_rows_have_gradients_of_zero(groups):
    """[batch, 0, dim] with a gate for each of the batch."""
    x = torch.empty(groups, 0, 64, device="cuda")
    w, gate = torch.ones(64, device="cuda"), torch.ones(groups, 64, device="cuda")
    r, h, stats = lm.norm_residual_forward(x, x, w, post_weight=w, gate=gate)
    assert r.shape == h.shape == x.shape
    got = lm.norm_residual_backward(None, h, x, x, w, stats, post_weight=w, gate=gate)
    assert got["gate"].shape == gate.shape and not bool(got["gate"].any()) and not bool(got["pre_weight"].any()) and not bool(got["post_weight"].any())
