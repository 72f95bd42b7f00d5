"""Sizes beyond one launch's first dimension (2^32 threads): every row is still worked on."""
import pytest
import torch

import stquant_lm as lm

pytestmark = pytest.mark.gpu


def test_distillation_of_more_rows_than_a_launch_dimension():
    n, v = (1 << 24) + 300, 8
    z = torch.zeros(n, v, dtype=torch.bfloat16, device="cuda")
    ids = torch.full((n, 1), 3, dtype=torch.int32, device="cuda")
    ids[-1], ids[1 << 21], ids[(1 << 24) + 1] = 5, 6, 7
    t = torch.zeros(n, 1, dtype=torch.bfloat16, device="cuda")
    loss, dz = lm.distill_loss_and_grad(z, t, ids, grad=1.0)
    _, stats = lm.distill_loss_forward(z, t, ids)
    two = lm.distill_loss_backward(1.0, z, t, ids, stats)
    # uniform over 8, certain of one: log 8, and 1/8 less the entry's 1
    assert float((loss - 2.0794415).abs().max()) < 1e-5
    want = torch.full((n, v), 0.125, dtype=torch.bfloat16, device="cuda")
    want.scatter_(1, ids.long(), -0.875)
    assert torch.equal(dz, want) and torch.equal(two, want)


def test_attention_gradients_of_more_rows_than_a_launch_dimension():
    """A window of one key: out is v, dv is dout and the scores have no gradients, all exactly."""
    b, h, t, d = 1, 65535, 4099, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randint(-8, 9, (b, h, t, d), dtype=torch.int8, device="cuda", generator=g).to(torch.bfloat16)
    do = x + 1
    out, lse = lm.attention_forward(x, x, x, window=1)
    assert torch.equal(out, x)
    dq, dk, dv = lm.attention_backward(do, x, x, x, out, lse, window=1)
    assert torch.equal(dv, do)
    assert not bool(dq.any()) and not bool(dk.any())


def test_lookup_of_more_rows_than_a_launch_dimension():
    n, vocab, dim = (1 << 24) + 77, 5, 515
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.randn(vocab, dim, device="cuda", generator=g).to(torch.bfloat16)
    tok = torch.arange(n, device="cuda", dtype=torch.int32) % vocab
    out = lm.embedding_forward(tok, w)
    for a in range(0, n, 1 << 21):
        b = min(n, a + (1 << 21))
        assert torch.equal(out[a:b], w[tok[a:b].long()]), a
