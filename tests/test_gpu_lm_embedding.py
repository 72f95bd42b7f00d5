"""Embedding lookup with scaling and its dense gradient against 64 bits: types, odd widths, strides, repeated
tokens, padding, tokens outside the table, accumulation; the same bits on every call.

Tolerances: the lookup rounds the scaled value to fp32 and to the output's type; a gradient of n rows is n
fp32 additions and one multiplication, at most (n + 2) 2^-24 of the magnitudes added, and one rounding."""
import pytest
import torch

import lm_reference as ref
import stquant_lm as lm

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def grad_bound(tokens, vocab, mag):
    count = torch.bincount(tokens.reshape(-1).clamp(0, vocab - 1).long(), minlength=vocab).double()[:, None]
    return (count + 2) * 2.0 ** -24 * mag


@pytest.mark.parametrize("n,vocab,dim", [(1, 1, 1), (7, 11, 3), (64, 500, 64), (5, 50257, 768), (1000, 333, 129), (300, 97, 4096), (65, 40, 2056)])
@pytest.mark.parametrize("wdt,odt", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F16), (BF16, F32)])
def test_lookup(n, vocab, dim, wdt, odt):
    g = ref.gen(n + dim)
    w = ref.randn(g, vocab, dim, std=0.02, dtype=wdt)
    tok = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    for scale in (1.0, dim ** 0.5):
        want = w.double()[tok] * float(torch.tensor(scale))
        ref.within("out", lm.embedding_forward(tok, w, scale=scale, dtype=odt), want, 2.0 ** -24 * want.abs())
    got = lm.embedding_forward(tok.int().view(1, n), w, dtype=odt)
    assert got.shape == (1, n, dim) and torch.equal(got[0], lm.embedding_forward(tok, w, dtype=odt))


@pytest.mark.parametrize("n,vocab,dim", [(1, 3, 8), (17, 5, 24), (200, 7, 100), (4097, 997, 65), (3000, 40000, 256), (2048, 1, 40), (5000, 300, 768)])
@pytest.mark.parametrize("gdt,wdt", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F32, BF16)])
def test_gradient(n, vocab, dim, gdt, wdt):
    g = ref.gen(n + vocab)
    tok = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    tok[: n // 2] = tok[: n // 2] % max(1, vocab // 50)          # half the tokens from few rows: runs over many waves
    grad = ref.randn(g, n, dim, dtype=gdt)
    want, mag = ref.embedding_grad(grad, tok, vocab, scale=1.5, padding=2)
    got = lm.embedding_backward(grad, tok, vocab, scale=1.5, padding_idx=2, dtype=wdt)
    ref.within("dweight", got, want, grad_bound(tok, vocab, mag))
    assert torch.equal(got, lm.embedding_backward(grad, tok.int(), vocab, scale=1.5, padding_idx=2, dtype=wdt))


@pytest.mark.parametrize("n", [40_000, 140_001])
def test_one_token_for_every_position_and_a_long_list(n):
    """A single row that gathers every gradient, and more entries than a wave keeps in LDS."""
    g = ref.gen(n)
    grad = ref.randn(g, n, 16)
    tok = torch.full((n,), 5, device="cuda")
    want, mag = ref.embedding_grad(grad, tok, 9)
    ref.within("dweight", lm.embedding_backward(grad, tok, 9), want, grad_bound(tok, 9, mag))
    tok = torch.randint(0, 600, (n,), device="cuda", generator=g)
    want, mag = ref.embedding_grad(grad, tok, 600)
    ref.within("dweight", lm.embedding_backward(grad, tok, 600), want, grad_bound(tok, 600, mag))


def test_a_vocabulary_of_many_ranges():
    g = ref.gen(3)
    vocab = 300_001
    tok = torch.randint(0, vocab, (2000,), device="cuda", generator=g)
    grad = ref.randn(g, 2000, 8)
    want, mag = ref.embedding_grad(grad, tok, vocab)
    ref.within("dweight", lm.embedding_backward(grad, tok, vocab), want, grad_bound(tok, vocab, mag))


def test_tokens_outside_the_table():
    w = ref.randn(ref.gen(0), 10, 24)
    tok = torch.tensor([3, -1, 10, 9, 2 ** 40, -(2 ** 40)], device="cuda")
    out = lm.embedding_forward(tok, w)
    assert torch.equal(out[[0, 3]], w[[3, 9]]) and bool(out[[1, 2, 4, 5]].isnan().all())
    grad = torch.ones(6, 24, device="cuda")
    want, _ = ref.embedding_grad(grad, tok, 10)
    assert torch.equal(lm.embedding_backward(grad, tok, 10).double(), want)


def test_empty_calls():
    w = ref.randn(ref.gen(0), 10, 24)
    tok = torch.empty(0, dtype=torch.int64, device="cuda")
    assert lm.embedding_forward(tok, w).shape == (0, 24)
    assert torch.equal(lm.embedding_backward(torch.empty(0, 24, device="cuda"), tok, 10), torch.zeros(10, 24, device="cuda"))


@pytest.mark.parametrize("dim,pad,shift", [(96, 32, 0), (64, 5, 0), (64, 8, 1), (33, 0, 3)])
def test_views(dim, pad, shift):
    """Rows that lie apart, at any offset: tables and gradients as parts of larger buffers."""
    g = ref.gen(dim + shift)
    w = ref.randn(g, 50 * (dim + pad) + shift, dtype=BF16)[shift:].view(50, dim + pad)[:, :dim]
    tok = torch.randint(0, 50, (333,), device="cuda", generator=g)
    assert torch.equal(lm.embedding_forward(tok, w), w[tok])
    grad = ref.randn(g, 333 * (dim + pad) + shift, dtype=BF16)[shift:].view(333, dim + pad)[:, :dim]
    want, mag = ref.embedding_grad(grad, tok, 50)
    ref.within("dweight", lm.embedding_backward(grad, tok, 50), want, grad_bound(tok, 50, mag))
    assert torch.equal(lm.embedding_backward(grad.t().contiguous().t(), tok, 50), lm.embedding_backward(grad, tok, 50))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_accumulation(dtype):
    g = ref.gen(8)
    tok = torch.randint(0, 20, (4, 25), device="cuda", generator=g)
    grad = ref.randn(g, 4, 25, 48, dtype=dtype)
    buf = ref.randn(g, 40, 48 + 16, dtype=dtype)
    had = buf.clone()
    out = lm.embedding_backward(grad, tok, 40, out=buf[:, :48])
    assert out.data_ptr() == buf.data_ptr() and torch.equal(buf[:, 48:], had[:, 48:])
    want, mag = ref.embedding_grad(grad, tok, 40)
    ref.within("dweight", buf[:, :48], had[:, :48].double() + want, grad_bound(tok, 40, mag) + 2.0 ** -23 * (mag + had[:, :48].abs()))
    assert torch.equal(buf[20:, :48], had[20:, :48])


def test_nan_and_inf_stay_with_their_token():
    tok = torch.tensor([1, 2, 2, 3], device="cuda")
    grad = torch.ones(4, 64, device="cuda")
    grad[0, 5], grad[1, 7] = float("nan"), float("inf")
    got = lm.embedding_backward(grad, tok, 6)
    want, mag = ref.embedding_grad(grad, tok, 6)
    ref.within("dweight", got, want, 0 * mag)


def test_autograd_and_differences():
    g = ref.gen(4)
    w = ref.randn(g, 30, 40).requires_grad_(True)
    tok = torch.randint(0, 30, (3, 20), device="cuda", generator=g)
    up = ref.randn(g, 3, 20, 40)
    (lm.embedding(tok, w, scale=3.0, padding_idx=int(tok[0, 0])) * up).sum().backward()
    want, mag = ref.embedding_grad(up, tok, 30, scale=3.0, padding=int(tok[0, 0]))
    ref.within("dweight", w.grad, want, grad_bound(tok, 30, mag))
    d = ref.randn(g, 30, 40).double()
    d[int(tok[0, 0])] = 0
    num = ref.differences(lambda x: (x[tok] * 3.0 * up.double()).sum(), [w.detach()], 0, d, 1e-3)
    assert abs(float(num) - float((w.grad.double() * d).sum())) <= float((grad_bound(tok, 30, mag) * d.abs()).sum()) + 1e-8


def test_a_captured_call_replays():
    g = ref.gen(6)
    w, grad = ref.randn(g, 70, 64), ref.randn(g, 90, 64)
    tok = torch.randint(0, 70, (90,), device="cuda", generator=g)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        lm.embedding_forward(tok, w), lm.embedding_backward(grad, tok, 70)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, dw = lm.embedding_forward(tok, w), lm.embedding_backward(grad, tok, 70)
    for step in range(3):
        tok.copy_(torch.randint(0, 70, (90,), device="cuda", generator=g))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, lm.embedding_forward(tok, w)) and torch.equal(dw, lm.embedding_backward(grad, tok, 70)), step
