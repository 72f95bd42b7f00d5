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


def step(monkeypatch, model, weight):
    """A step whose loss has a gradient of ones: the gradient of ``weight``."""
    monkeypatch.setattr(dp.lm, "distill_loss_and_grad", lambda z, *targets, out, **k: (z.sum(-1), out.fill_(1.0)))
    weight.grad = None
    loss = dp.step_loss(model, torch.tensor([[0, 2, 1]]), (), temperature=1.0, alpha=0.5, balance=0.25)
    assert loss.shape == ()
    return weight.grad


class Table(torch.nn.Module):
    """Logits from a table; with ``sparse`` a load term as the sparse decoder's."""

    def __init__(self, sparse=False):
        super().__init__()
        self.rows, self.sparse = torch.nn.Parameter(torch.arange(12.0).view(3, 4)), sparse

    def forward(self, tokens):
        if self.sparse:
            self.uneven = 8.0 * self.rows[0, 0]
        return self.rows[tokens] * 2.0


class Wrapped(torch.nn.Module):
    """As the wrappers for several ranks: the model is ``module``, and none of its attributes is passed on."""

    def __init__(self, module):
        super().__init__()
        self.module = module

    def forward(self, tokens):
        return self.module(tokens)


def test_a_step_takes_models_without_a_load_term(monkeypatch):
    table = Table()
    for model in (table, Wrapped(table), lambda t: table(t)):
        assert torch.equal(step(monkeypatch, model, table.rows), torch.full((3, 4), 2.0))


def test_a_step_finds_the_load_term_in_a_wrapped_model(monkeypatch):
    table = Table(sparse=True)
    want = torch.full((3, 4), 2.0)
    want[0, 0] += 0.25 * 8.0
    for model in (table, Wrapped(table)):
        assert torch.equal(step(monkeypatch, model, table.rows), want)
        assert not table.uneven.requires_grad


def test_a_decoder_from_before_the_sparse_mlp_is_dense():
    """One that was saved whole has no such attributes of its own."""
    old = dp.Decoder(40, 16, 1, 2, device="cpu")
    for name in ("experts", "top_experts"):
        del old.__dict__[name]
    assert old.experts == 0 and old.uneven is None
