"""The example's model without a GPU: the arguments and attributes that calls from before the sparse MLP rely on."""
import torch

import distill_pretrain as dp


def test_positional_arguments_mean_what_they_meant():
    """(vocab, n_embd, n_layer, n_head, n_kv, window, sinks, seed, device), the sparse MLP's by name alone."""
    a, b = dp.Decoder(40, 16, 1, 2, 0, 4, 1, 7, "cpu"), dp.Decoder(vocab=40, n_embd=16, n_layer=1, n_head=2, window=4, sinks=1, seed=7, device="cpu")
    assert a.experts == b.experts == 0 and (a.window, a.sinks) == (4, 1)
    assert all(torch.equal(x, y) for x, y in zip(a.parameters(), b.parameters(), strict=True))
    sparse = dp.Decoder(40, 16, 1, 2, 0, 4, 1, 7, "cpu", experts=3, top_experts=1, expert_width=24)
    assert sparse.up[0].shape == (3, 24, 16) and sparse.top_experts == 1 and torch.equal(sparse.wte, a.wte)
