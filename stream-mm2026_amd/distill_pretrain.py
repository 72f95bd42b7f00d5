"""Training a small decoder from a teacher's top logits with the low-bit optimizer.

The operators of ``stquant_lm`` as a training step uses them together: the tokens enter through
``embedding`` (scaled, its table tied to the output layer), every block mixes them with ``attention``
over a window of the last positions and a few first ones, ``norm_residual`` carries the residual stream
(a norm after each block, a gate per channel, the next block's norm) and ``distill_loss_and_grad`` turns
the logits into the loss's gradient in place.  With ``experts`` the MLP is a sparse one: ``route`` sends each
position to a few experts, ``expert_product`` and ``expert_combine`` compute them, and a small loss keeps them evenly
loaded; nearly all parameters are then the experts', whose optimizer state the low-bit codes shrink.  The
parameters are fp32 and stepped by the fused MDQ optimizer, their gradients first clipped to a global norm where one is
given; activations are bfloat16.  The dense matrix products are torch's.

The teacher is a frozen model of the same kind; its top ``k`` logits per position and the next tokens are
the targets.  Tokens are synthetic: uniform over the first ``vocab_used`` ids, from one seeded generator.

Usage::

    python distill_pretrain.py --steps 100 --window 256 --sinks 4
    python distill_pretrain.py --experts 8 --top-experts 2 --expert-width 1536 --max-grad-norm 1.0
"""
from __future__ import annotations

import argparse
import json
import math
import os
import sys
import time

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
if _HERE not in sys.path:
    sys.path.insert(0, _HERE)

import stquant_lm as lm  # noqa: E402
from gpt2_pretrain import OPTIMIZERS, VOCAB, build_optimizer  # noqa: E402


class Decoder(torch.nn.Module):
    """A decoder with norms before and after each attention and MLP block (GPT-2 small's sizes by default)."""
    experts, uneven = 0, None            # (a dense one)

    def __init__(self, vocab: int = VOCAB, n_embd: int = 768, n_layer: int = 12, n_head: int = 12, n_kv: int = 0,
                 window: int = 0, sinks: int = 0, seed: int = 42, device="cuda:0", *, experts: int = 0, top_experts: int = 2,
                 expert_width: int = 0):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        self.experts, self.top_experts = experts, top_experts
        self.n_layer, self.n_head, self.n_kv, self.dim = n_layer, n_head, n_kv or n_head, n_embd // n_head
        self.window, self.sinks = window, sinks

        def weight(*shape, std=0.02):
            return torch.nn.Parameter((torch.randn(*shape, generator=g) * std).to(device))

        def ones(value=1.0):
            return torch.nn.Parameter(torch.full((n_embd,), value, device=device))

        self.wte = weight(vocab, n_embd)
        kv = self.n_kv * self.dim
        out_std = 0.02 / math.sqrt(2 * n_layer)
        self.qkv = torch.nn.ParameterList([weight(n_embd + 2 * kv, n_embd) for _ in range(n_layer)])
        self.proj = torch.nn.ParameterList([weight(n_embd, n_embd, std=out_std) for _ in range(n_layer)])
        width = expert_width or 4 * n_embd
        of = (experts,) if experts else ()
        self.up = torch.nn.ParameterList([weight(*of, width, n_embd) for _ in range(n_layer)])
        self.down = torch.nn.ParameterList([weight(*of, n_embd, width, std=out_std) for _ in range(n_layer)])
        if experts:
            self.router = torch.nn.ParameterList([weight(experts, n_embd) for _ in range(n_layer)])
        # the first norm, then for each of the 2 n_layer blocks: the norm behind it, its gate, the next norm
        self.first = ones()
        self.post = torch.nn.ParameterList([ones() for _ in range(2 * n_layer)])
        self.gate = torch.nn.ParameterList([ones(1.0 / math.sqrt(2 * n_layer)) for _ in range(2 * n_layer)])
        self.pre = torch.nn.ParameterList([ones() for _ in range(2 * n_layer)])

    def mix(self, h: torch.Tensor, layer: int, key_mask=None) -> torch.Tensor:
        b, t, d = h.shape
        kv = self.n_kv * self.dim
        q, k, v = torch.nn.functional.linear(h, self.qkv[layer].to(h.dtype)).split([d, kv, kv], -1)
        heads = lambda x: x.view(b, t, -1, self.dim).transpose(1, 2)  # noqa: E731
        o = lm.attention(heads(q), heads(k), heads(v), window=self.window, sinks=self.sinks, key_mask=key_mask)
        return torch.nn.functional.linear(o.transpose(1, 2).reshape(b, t, d), self.proj[layer].to(h.dtype))

    def mlp(self, h: torch.Tensor, layer: int) -> torch.Tensor:
        u = torch.nn.functional.gelu(torch.nn.functional.linear(h, self.up[layer].to(h.dtype)), approximate="tanh")
        return torch.nn.functional.linear(u, self.down[layer].to(h.dtype))

    def sparse(self, h: torch.Tensor, layer: int):
        """The sparse MLP, and how unevenly its experts are loaded (1: evenly)."""
        logits = torch.nn.functional.linear(h.float(), self.router[layer])
        weights, ids, load = lm.route(logits, self.top_experts, renormalize=True)
        plan = lm.expert_plan(ids, self.experts)
        u = torch.nn.functional.gelu(lm.expert_product(h, self.up[layer].to(h.dtype), plan, gather=True), approximate="tanh")
        y = lm.expert_product(u, self.down[layer].to(h.dtype), plan)
        share = plan.offsets.diff() / ids.numel()
        uneven = self.experts * (share * load).sum() * (self.top_experts / ids.numel())
        return lm.expert_combine(y, weights, plan), uneven

    def forward(self, tokens: torch.Tensor, key_mask=None) -> torch.Tensor:
        """The logits [batch, time, vocab] in bfloat16.  ``uneven`` then holds the layers' mean of how unevenly the experts
        are loaded (sparse MLPs; None otherwise)."""
        self.uneven = None
        x = lm.embedding(tokens, self.wte, scale=math.sqrt(self.wte.shape[1]), dtype=torch.bfloat16)
        h = torch.nn.functional.rms_norm(x, x.shape[-1:], self.first.to(x.dtype), 1e-5)
        for i in range(2 * self.n_layer):
            if i % 2 == 0:
                y = self.mix(h, i // 2, key_mask)
            elif self.experts:
                y, uneven = self.sparse(h, i // 2)
                self.uneven = uneven / self.n_layer + (0.0 if self.uneven is None else self.uneven)
            else:
                y = self.mlp(h, i // 2)
            x, h = lm.norm_residual(x, y, self.pre[i], post_weight=self.post[i], gate=self.gate[i], eps=1e-5)
        return torch.nn.functional.linear(h, self.wte.to(h.dtype))


@torch.no_grad()
def teach(teacher: Decoder, tokens: torch.Tensor, k: int):
    """The teacher's top ``k`` logits and their ids, [batch, time, k]."""
    return torch.topk(teacher(tokens), k, dim=-1)


def step_loss(model: Decoder, tokens: torch.Tensor, targets, *, temperature: float, alpha: float, balance: float = 0.01) -> torch.Tensor:
    """Forward and backward of one batch: the mean loss; the gradients are in the parameters, with ``balance`` times
    those of how unevenly experts are loaded, where the model (or the ``module`` that it wraps) says so."""
    logits = model(tokens)
    labels = torch.full_like(tokens, -100)
    labels[:, :-1] = tokens[:, 1:]
    # the gradient takes the logits' place: nothing else needs them
    z = logits.detach()
    loss, dz = lm.distill_loss_and_grad(z, *targets, grad=1.0 / tokens.numel(), labels=labels, temperature=temperature, alpha=alpha, out=z)
    inner = model if hasattr(model, "uneven") else getattr(model, "module", model)      # (as wrappers for several ranks hold it)
    uneven = getattr(inner, "uneven", None)
    if uneven is None:
        logits.backward(dz)
    else:
        torch.autograd.backward([logits, balance * uneven], [dz, None])
        inner.uneven = uneven.detach()         # (the number: its graph would live until the next call)
    return loss.mean()


def train(optimizer_name: str = "MDQAdamW-Simple-FusedIO", *, steps: int = 100, warmup: int = 3, batch: int = 8, seq_len: int = 1024,
          lr: float = 2e-4, bits=4, rounding: str = "stochastic", k: int = 64, temperature: float = 2.0, alpha: float = 0.7,
          vocab: int = VOCAB, vocab_used: int = VOCAB, n_layer: int = 12, n_embd: int = 768, n_head: int = 12, n_kv: int = 0,
          window: int = 256, sinks: int = 4, experts: int = 0, top_experts: int = 2, expert_width: int = 0, balance: float = 0.01,
          max_grad_norm: float = 0.0, data_seed: int = 1234, device="cuda:0", log_every: int = 0) -> dict:
    """``steps`` measured steps after ``warmup`` ones; returns losses and times.  ``max_grad_norm`` > 0: the gradients are
    clipped to that norm before each optimizer step."""
    dev = torch.device(device)
    shape = dict(vocab=vocab, n_embd=n_embd, n_layer=n_layer, n_head=n_head, n_kv=n_kv, window=window, sinks=sinks, experts=experts,
                 top_experts=top_experts, expert_width=expert_width, device=dev)
    model, teacher = Decoder(seed=42, **shape), Decoder(seed=7, **shape)
    opt = build_optimizer(optimizer_name, model, lr, n_layer, batch, bits=bits, rounding=rounding)
    gen = torch.Generator(device=dev).manual_seed(data_seed)
    losses, ms = [], []
    for it in range(warmup + steps):
        tokens = torch.randint(0, vocab_used, (batch, seq_len), device=dev, generator=gen)
        values, ids = teach(teacher, tokens, k)
        torch.cuda.synchronize(dev)
        t0 = time.perf_counter()
        loss = step_loss(model, tokens, (values, ids), temperature=temperature, alpha=alpha, balance=balance)
        if max_grad_norm > 0:
            lm.clip_grads([p.grad for p in model.parameters() if p.grad is not None], max_grad_norm)
        opt.step()
        opt.zero_grad(set_to_none=True)
        torch.cuda.synchronize(dev)
        if it >= warmup:
            ms.append((time.perf_counter() - t0) * 1e3)
            losses.append(float(loss))
            if log_every and len(losses) % log_every == 0:
                print(f"[distill] step {len(losses)}/{steps} loss {losses[-1]:.4f} {ms[-1]:.1f} ms", file=sys.stderr, flush=True)
    return {"Opt": optimizer_name, "Params": sum(p.numel() for p in model.parameters()), "First_Loss": losses[0], "Final_Loss": losses[-1],
            "Avg_Step_ms": sum(ms) / len(ms), "Tokens_per_s": batch * seq_len * len(ms) / sum(ms) * 1e3, "Losses": losses}


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--optimizer", choices=OPTIMIZERS, default="MDQAdamW-Simple-FusedIO")
    ap.add_argument("--steps", type=int, default=100)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--seq-len", type=int, default=1024)
    ap.add_argument("--lr", type=float, default=2e-4)
    ap.add_argument("--top-k", type=int, default=64)
    ap.add_argument("--temperature", type=float, default=2.0)
    ap.add_argument("--alpha", type=float, default=0.7)
    ap.add_argument("--window", type=int, default=256)
    ap.add_argument("--sinks", type=int, default=4)
    ap.add_argument("--kv-heads", type=int, default=0)
    ap.add_argument("--experts", type=int, default=0, help="experts of a sparse MLP (0: a dense one)")
    ap.add_argument("--top-experts", type=int, default=2)
    ap.add_argument("--expert-width", type=int, default=0)
    ap.add_argument("--balance", type=float, default=0.01)
    ap.add_argument("--max-grad-norm", type=float, default=0.0)
    a = ap.parse_args(argv)
    res = train(a.optimizer, steps=a.steps, batch=a.batch, seq_len=a.seq_len, lr=a.lr, k=a.top_k, temperature=a.temperature, alpha=a.alpha,
                window=a.window, sinks=a.sinks, n_kv=a.kv_heads, experts=a.experts, top_experts=a.top_experts, expert_width=a.expert_width,
                balance=a.balance, max_grad_norm=a.max_grad_norm, log_every=25)
    print(json.dumps({k: v for k, v in res.items() if k != "Losses"}))


if __name__ == "__main__":
    main()
