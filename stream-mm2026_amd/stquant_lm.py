"""Transformer operators for models trained with the low-bit optimizer, on hand-written HIP kernels.

What a training step runs around the optimizer, each with its gradient:

``embedding``      table lookup with scaling; the table's dense gradient by sorted tokens
``norm_residual``  the norms before and after a block, fused with its gate and the residual sum
``attention``      causal attention over a window of the last keys and a few first ones (sinks)
``distill_loss``   learning from a teacher's top logits, mixed with the labels' cross-entropy

The plain names are differentiable (``torch.autograd``), once: a second derivative raises.  The
``*_forward`` / ``*_backward`` pairs and ``distill_loss_and_grad`` are the calls beneath them, for
training loops that hold their own buffers.
Everything runs on the current stream of the tensors' device through the C ABI of
``include/stquant_lm.h``; nothing synchronises, so calls can be captured into a graph.  As with torch's
own operators, a tensor used on another stream than the one it was allocated on is the caller's to keep
alive.  There is no CPU or eager fallback.  Sums, softmax statistics and norms are fp32 whatever the
tensors' type, and the same call gives the same bits every time.
"""
from __future__ import annotations

import os
import struct
import sys
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

_HERE = os.path.dirname(os.path.abspath(__file__))
if _HERE not in sys.path:
    sys.path.insert(0, _HERE)

from mdq_hip import _capi  # noqa: E402
from mdq_hip._capi import check, lm_lib  # noqa: E402

__all__ = [
    "embedding", "embedding_forward", "embedding_backward",
    "norm_residual", "norm_residual_forward", "norm_residual_backward",
    "attention", "attention_forward", "attention_backward",
    "distill_loss", "distill_loss_forward", "distill_loss_backward", "distill_loss_and_grad",
]

_FLOATS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_INDEXES = {torch.int64: 9, torch.int32: 7}
# The argument structs of stquant_lm.h, every field 8 bytes (packing them costs 1 us; ctypes fields 0.2 us each).
_EMBED = struct.Struct("@Qqqqq Qqq Qq d")
_EMBED_GRAD = struct.Struct("@Qqqqq Qqq Qqq qq Qq d")
_NORM = struct.Struct("@4q 2Q2q 5Q 2q 2d 3Q 2Q2q 7Q Qq")
_ATTN = struct.Struct("@9q d 4q4q4q4q Qq Q 4q4q4q4q Qq")
_DISTILL = struct.Struct("@3q Qq Qq Qqq Qq 2d 2Q Q Qq")


def _fail(msg: str):
    raise RuntimeError(msg)


def _float_code(name: str, t: torch.Tensor) -> int:
    code = _FLOATS.get(t.dtype)
    if code is None:
        _fail(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _index_code(name: str, t: torch.Tensor) -> int:
    code = _INDEXES.get(t.dtype)
    if code is None:
        _fail(f"{name} must be int64 or int32, got {t.dtype}")
    return code


def _same_device(first: torch.Tensor, **others: Optional[torch.Tensor]) -> None:
    dev = first.get_device()
    if dev < 0:
        _fail("tensors must be CUDA")
    for name, t in others.items():
        if t is not None and t.get_device() != dev:
            _fail(f"{name} must be on {first.device}, got {t.device}")


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _call(dev: torch.device, fn, packed: bytes) -> None:
    _capi.launch(dev, fn, packed)


def _size(fn, packed: bytes) -> int:
    n = fn(packed)
    if n < 0:
        check(_capi.STQ_ERR_INVALID)
    return n


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """``t`` as [rows, width] with dense rows (a view wherever its strides allow one)."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    return t if t.stride(1) == 1 or width == 1 else t.contiguous()


def _written(*tensors: torch.Tensor) -> None:
    """Tensors of the caller that a call has written count as changed in place: autograd then refuses to use one that
    another operation saved."""
    for t in tensors:
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _workspace(nbytes: int, dev: torch.device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


# ---------------------------------------------------------------- embedding
def embedding_forward(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0,
                      dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``scale * weight[tokens]`` as [*tokens.shape, dim] in ``dtype`` (default: the weight's; rounded once).

    A token outside the table gives a row of NaN."""
    ic = _index_code("tokens", tokens)
    wc = _float_code("weight", weight)
    if weight.dim() != 2:
        _fail(f"weight must be [vocab, dim], got {tuple(weight.shape)}")
    _same_device(weight, tokens=tokens)
    if weight.stride(1) != 1 and weight.shape[1] != 1:
        _fail("weight must have dense rows")
    out = torch.empty((*tokens.shape, weight.shape[1]), dtype=dtype or weight.dtype, device=weight.device)
    oc = _float_code("out", out)
    tokens = tokens.contiguous()
    _call(weight.device, lm_lib().stq_embedding_forward,
          _EMBED.pack(tokens.data_ptr(), ic, tokens.numel(), weight.shape[0], weight.shape[1], weight.data_ptr(), wc,
                      weight.stride(0), out.data_ptr(), oc, float(scale)))
    return out


def embedding_backward(grad: torch.Tensor, tokens: torch.Tensor, num_embeddings: int, *, scale: float = 1.0,
                       padding_idx: Optional[int] = None, dtype: Optional[torch.dtype] = None,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The dense gradient [num_embeddings, dim] of the table: ``scale`` times the sum of each token's
    rows of ``grad``, added in the order of the tokens in fp32.

    ``dtype`` defaults to the grad's.  ``out``: added to what it holds, rows of no token untouched
    (gradient accumulation, or a table shared with the output layer).  ``padding_idx`` takes none."""
    ic = _index_code("tokens", tokens)
    gc = _float_code("grad", grad)
    if grad.dim() < 1 or grad.shape[:-1] != tokens.shape:
        _fail(f"grad must be {(*tokens.shape, 'dim')}, got {tuple(grad.shape)}")
    dim = grad.shape[-1]
    _same_device(grad, tokens=tokens, out=out)
    if padding_idx is not None and padding_idx < 0:
        padding_idx += num_embeddings
    g = _rows(grad, dim) if dim else grad
    tokens = tokens.contiguous()
    dw = out
    if dw is None:
        dw = torch.empty((num_embeddings, dim), dtype=dtype or grad.dtype, device=grad.device)
    elif tuple(dw.shape) != (num_embeddings, dim) or (dw.stride(1) != 1 and dim != 1):
        _fail(f"out must be [{num_embeddings}, {dim}] with dense rows")
    elif dtype is not None and dw.dtype != dtype:
        _fail(f"out must be {dtype}, got {dw.dtype}")
    dc = _float_code("dweight", dw)
    L = lm_lib()
    args = [tokens.data_ptr(), ic, tokens.numel(), num_embeddings, dim, g.data_ptr(), gc, g.stride(0), dw.data_ptr(), dc, dw.stride(0),
            -1 if padding_idx is None else padding_idx, int(out is not None), 0, 0, float(scale)]
    ws = _workspace(_size(L.stq_embedding_grad_workspace, _EMBED_GRAD.pack(*args)), grad.device)
    args[13:15] = ws.data_ptr(), ws.numel()
    _call(grad.device, L.stq_embedding_backward, _EMBED_GRAD.pack(*args))
    if out is not None:
        _written(out)
    return dw


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding_idx, dtype):
        ctx.save_for_backward(tokens)
        ctx.args = (weight.shape[0], scale, padding_idx, weight.dtype)
        return embedding_forward(tokens, weight, scale=scale, dtype=dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (tokens,) = ctx.saved_tensors
        n, scale, padding_idx, dtype = ctx.args
        dw = embedding_backward(grad, tokens, n, scale=scale, padding_idx=padding_idx, dtype=dtype)
        return None, dw, None, None, None


def embedding(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, padding_idx: Optional[int] = None,
              dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``scale * weight[tokens]``, differentiable in ``weight`` (a dense gradient of its type)."""
    return _Embedding.apply(tokens, weight, scale, padding_idx, dtype)


# ---------------------------------------------------------------- residual norms
_KINDS = {"rms": 0, "layer": 1}


def _norm_args(x, block, pre_weight, pre_bias, post_weight, post_bias, gate, residual_scale, eps, kind):
    """The checked operands, x and block as rows, and the struct's leading fields."""
    if kind not in _KINDS:
        raise ValueError(f"kind must be 'rms' or 'layer', got {kind!r}")
    xc = _float_code("x", x)
    if x.dim() < 1 or x.shape != block.shape:
        _fail(f"x and block must have one shape, got {tuple(x.shape)} and {tuple(block.shape)}")
    if block.dtype != x.dtype:
        _fail(f"block must be {x.dtype}, got {block.dtype}")
    dim = x.shape[-1]
    _same_device(x, block=block, pre_weight=pre_weight, pre_bias=pre_bias, post_weight=post_weight, post_bias=post_bias, gate=gate)
    wc = _float_code("pre_weight", pre_weight)
    for name, w in (("pre_weight", pre_weight), ("pre_bias", pre_bias), ("post_weight", post_weight), ("post_bias", post_bias)):
        if w is not None and (w.shape != (dim,) or w.dtype != pre_weight.dtype or not w.is_contiguous()):
            _fail(f"{name} must be a dense [{dim}] of {pre_weight.dtype}, got {tuple(w.shape)} of {w.dtype}")
    if kind == "rms" and (pre_bias is not None or post_bias is not None):
        _fail("RMS norms have no bias")
    groups = 1
    if gate is not None:
        if gate.shape[-1:] != (dim,) or gate.dtype != pre_weight.dtype or not gate.is_contiguous():
            _fail(f"gate must be a dense [{dim}] or [groups, {dim}] of {pre_weight.dtype}, got {tuple(gate.shape)} of {gate.dtype}")
        groups = gate.numel() // dim
    x, block = _rows(x, dim), _rows(block, dim)
    n = x.shape[0]
    head = (n, dim, xc, wc, x.data_ptr(), block.data_ptr(), x.stride(0), block.stride(0), pre_weight.data_ptr(), _ptr(pre_bias),
            _ptr(post_weight), _ptr(post_bias), _ptr(gate), groups, _KINDS[kind], float(residual_scale), float(eps))
    return x, block, head


def norm_residual_forward(x: torch.Tensor, block: torch.Tensor, pre_weight: torch.Tensor, *, pre_bias: Optional[torch.Tensor] = None,
                          post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                          gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0, eps: float = 1e-5, kind: str = "rms"):
    """``(r, h, stats)``: the residual stream behind a block and the norm of it that the next block reads.

    ``n1 = norm(block; post_weight, post_bias)`` (``block`` itself where ``post_weight`` is None),
    ``r = residual_scale * x + gate * n1``, ``h = norm(r; pre_weight, pre_bias)``.  ``kind``: ``"rms"`` or
    ``"layer"``.  ``gate``: [dim], or [groups, dim] for equal runs of rows ([batch, dim] gates [batch, time, dim]).
    Widths of 8 to 8192.  ``stats`` goes to the backward call."""
    shape = x.shape
    xr, br, head = _norm_args(x, block, pre_weight, pre_bias, post_weight, post_bias, gate, residual_scale, eps, kind)
    r = torch.empty(shape, dtype=x.dtype, device=x.device)
    h = torch.empty_like(r)
    stats = torch.empty((xr.shape[0], 4), dtype=torch.float32, device=x.device)
    _call(x.device, lm_lib().stq_norm_residual_forward,
          _NORM.pack(*head, stats.data_ptr(), r.data_ptr(), h.data_ptr(), *(0,) * 13))
    return r, h, stats


def norm_residual_backward(dr: Optional[torch.Tensor], dh: torch.Tensor, x: torch.Tensor, block: torch.Tensor, pre_weight: torch.Tensor,
                           stats: torch.Tensor, *, pre_bias: Optional[torch.Tensor] = None, post_weight: Optional[torch.Tensor] = None,
                           post_bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0,
                           kind: str = "rms") -> dict:
    """The gradients of ``x``, ``block`` and whichever of the weights, biases and gate are given, by name.

    ``dr`` and ``dh`` are the gradients of ``r`` and ``h`` (``dr`` None: zeros)."""
    xr, br, head = _norm_args(x, block, pre_weight, pre_bias, post_weight, post_bias, gate, residual_scale, 0.0, kind)
    dim = xr.shape[1]
    _same_device(x, dr=dr, dh=dh, stats=stats)
    for name, t in (("dr", dr), ("dh", dh)):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            _fail(f"{name} must be {tuple(x.shape)} of {x.dtype}, got {tuple(t.shape)} of {t.dtype}")
    if stats.dtype != torch.float32 or stats.shape != (xr.shape[0], 4) or not stats.is_contiguous():
        _fail(f"stats must be the forward call's [{xr.shape[0]}, 4]")
    dhr = _rows(dh, dim)
    drr = None if dr is None else _rows(dr, dim)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    grads = {"x": dx, "block": torch.empty_like(dx)}
    for name, w in (("pre_weight", pre_weight), ("pre_bias", pre_bias), ("post_weight", post_weight), ("post_bias", post_bias), ("gate", gate)):
        if w is not None:
            grads[name] = torch.empty_like(w)
    L = lm_lib()
    tail = [stats.data_ptr(), 0, 0, _ptr(drr), dhr.data_ptr(), 0 if drr is None else drr.stride(0), dhr.stride(0)]
    tail += [_ptr(grads.get(k)) for k in ("x", "block", "pre_weight", "pre_bias", "post_weight", "post_bias", "gate")]
    ws = _workspace(_size(L.stq_norm_residual_workspace, _NORM.pack(*head, *tail, 0, 0)), x.device)
    _call(x.device, L.stq_norm_residual_backward, _NORM.pack(*head, *tail, _ptr(ws), 0 if ws is None else ws.numel()))
    return grads


class _NormResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, block, pre_weight, pre_bias, post_weight, post_bias, gate, residual_scale, eps, kind):
        r, h, stats = norm_residual_forward(x, block, pre_weight, pre_bias=pre_bias, post_weight=post_weight, post_bias=post_bias,
                                            gate=gate, residual_scale=residual_scale, eps=eps, kind=kind)
        ctx.save_for_backward(x, block, pre_weight, pre_bias, post_weight, post_bias, gate, stats)
        ctx.args = (residual_scale, kind)
        ctx.set_materialize_grads(False)
        return r, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dr, dh):
        x, block, pre_weight, pre_bias, post_weight, post_bias, gate, stats = ctx.saved_tensors
        if dh is None:
            dh = torch.zeros_like(x)
        g = norm_residual_backward(dr, dh, x, block, pre_weight, stats, pre_bias=pre_bias, post_weight=post_weight, post_bias=post_bias,
                                   gate=gate, residual_scale=ctx.args[0], kind=ctx.args[1])
        return (*(g.get(k) for k in ("x", "block", "pre_weight", "pre_bias", "post_weight", "post_bias", "gate")), None, None, None)


def norm_residual(x: torch.Tensor, block: torch.Tensor, pre_weight: torch.Tensor, *, pre_bias: Optional[torch.Tensor] = None,
                  post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                  gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0, eps: float = 1e-5, kind: str = "rms"):
    """``(r, h)`` of :func:`norm_residual_forward`, differentiable in every tensor."""
    return _NormResidual.apply(x, block, pre_weight, pre_bias, post_weight, post_bias, gate, residual_scale, eps, kind)


# ---------------------------------------------------------------- attention
def _piecewise(t: torch.Tensor) -> torch.Tensor:
    """``t`` as the kernels read it: 16-byte pieces, dense along the head's elements (a copy if it is not)."""
    s = t.stride()
    if s[3] == 1 and not (s[0] % 8 or s[1] % 8 or s[2] % 8 or t.data_ptr() % 16):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _fields(t: Optional[torch.Tensor]):
    if t is None:
        return 0, 0, 0, 0
    s = t.stride()
    return t.data_ptr(), s[0], s[1], s[2]


def _attn_args(q, k, v, window, sinks, scale, key_mask):
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        _fail(f"q, k, v must be [batch, heads, positions, dim], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    b, h, t, d = q.shape
    hk, s = k.shape[1:3]
    if k.shape[0] != b or k.shape[3] != d:
        _fail(f"k and v must have q's batch and dim, got {tuple(q.shape)} and {tuple(k.shape)}")
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        _fail(f"q, k and v must all be bfloat16 or all float16, got {q.dtype}, {k.dtype}, {v.dtype}")
    if d % 8 or not 8 <= d <= 128:
        _fail(f"dim must be a multiple of 8 up to 128, got {d}")
    if hk == 0 or h % hk:
        _fail(f"heads ({h}) must be a multiple of the key heads ({hk})")
    if t > s:
        _fail(f"{t} positions cannot be the last of {s} keys")
    _same_device(q, k=k, v=v, key_mask=key_mask)
    if key_mask is not None:
        if key_mask.shape != (b, s) or key_mask.dtype not in (torch.bool, torch.uint8):
            _fail(f"key_mask must be a bool [{b}, {s}], got {tuple(key_mask.shape)} of {key_mask.dtype}")
        if key_mask.stride(1) != 1:
            key_mask = key_mask.contiguous()
    head = (_FLOATS[q.dtype], b, h, hk, t, s, d, int(window or 0), int(sinks), float(d ** -0.5 if scale is None else scale))
    return key_mask, head


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: Optional[int] = 0, sinks: int = 0,
                      scale: Optional[float] = None, key_mask: Optional[torch.Tensor] = None):
    """``(out, lse)`` of causal attention: q [batch, heads, rows, dim] over k, v [batch, key heads, keys, dim].

    The rows are the last positions of the keys: row i stands at ``p = keys - rows + i`` and sees key
    ``j <= p`` if ``p - j < window`` (0 or None: every one) or ``j < sinks``, and where ``key_mask``
    [batch, keys] is True.  A row that sees nothing is 0.  Consecutive ``heads / key heads`` heads share a
    key head.  bfloat16 or float16, dim a multiple of 8 up to 128; ``scale`` (> 0) defaults to dim ** -0.5.
    ``out`` is [batch, heads, rows, dim], laid out with the heads of a position side by side; ``lse``
    [batch, heads, rows] (fp32) goes to the backward call.  Weights are rounded to the tensors' type before
    their product with v."""
    key_mask, head = _attn_args(q, k, v, window, sinks, scale, key_mask)
    b, h, t, d = q.shape
    q, k, v = _piecewise(q), _piecewise(k), _piecewise(v)
    out = torch.empty((b, t, h, d), dtype=q.dtype, device=q.device).transpose(1, 2)
    lse = torch.empty((b, h, t), dtype=torch.float32, device=q.device)
    args = [*head, *_fields(q), *_fields(k), *_fields(v), *_fields(out), _ptr(key_mask), 0 if key_mask is None else key_mask.stride(0),
            lse.data_ptr(), *(0,) * 18]
    L = lm_lib()
    ws = _workspace(_size(L.stq_attention_forward_workspace, _ATTN.pack(*args)), q.device)
    if ws is not None:
        args[-2:] = ws.data_ptr(), ws.numel()
    _call(q.device, L.stq_attention_forward, _ATTN.pack(*args))
    return out, lse


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor, *,
                       window: Optional[int] = 0, sinks: int = 0, scale: Optional[float] = None,
                       key_mask: Optional[torch.Tensor] = None, grads=None):
    """``(dq, dk, dv)`` from the forward call's tensors; those of shared key heads are summed in fp32.
    Weights and score gradients are rounded to the tensors' type before their products (float16: scaled by
    powers of two that keep them among its normal numbers).

    ``grads``: three tensors to write them into (views of one buffer, for a joint projection), with dense
    elements, 16-byte aligned rows and no overlap."""
    key_mask, head = _attn_args(q, k, v, window, sinks, scale, key_mask)
    b, h, t, d = q.shape
    hk, s = k.shape[1:3]
    for name, x in (("dout", dout), ("out", out)):
        if x.shape != q.shape or x.dtype != q.dtype:
            _fail(f"{name} must be {tuple(q.shape)} of {q.dtype}, got {tuple(x.shape)} of {x.dtype}")
    if lse.shape != (b, h, t) or lse.dtype != torch.float32 or not lse.is_contiguous():
        _fail(f"lse must be the forward call's [{b}, {h}, {t}]")
    _same_device(q, dout=dout, out=out, lse=lse)
    q, k, v, out, dout = map(_piecewise, (q, k, v, out, dout))
    given = grads is not None
    if not given:
        grads = tuple(torch.empty((b, n, heads, d), dtype=q.dtype, device=q.device).transpose(1, 2) for n, heads in ((t, h), (s, hk), (s, hk)))
    else:
        for name, x, like in zip(("dq", "dk", "dv"), grads, (q, k, v)):
            if x.shape != like.shape or x.dtype != q.dtype or x.stride(3) != 1:
                _fail(f"{name} must be {tuple(like.shape)} of {q.dtype} with dense elements")
            _same_device(q, **{name: x})
    dq, dk, dv = grads
    args = [*head, *_fields(q), *_fields(k), *_fields(v), *_fields(out), _ptr(key_mask), 0 if key_mask is None else key_mask.stride(0),
            lse.data_ptr(), *_fields(dout), *_fields(dq), *_fields(dk), *_fields(dv), 0, 0]
    L = lm_lib()
    ws = _workspace(_size(L.stq_attention_backward_workspace, _ATTN.pack(*args)), q.device)
    if ws is not None:
        args[-2:] = ws.data_ptr(), ws.numel()
    _call(q.device, L.stq_attention_backward, _ATTN.pack(*args))
    if given:
        _written(dq, dk, dv)
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, scale, key_mask):
        out, lse = attention_forward(q, k, v, window=window, sinks=sinks, scale=scale, key_mask=key_mask)
        ctx.save_for_backward(q, k, v, out, lse, key_mask)
        ctx.args = dict(window=window, sinks=sinks, scale=scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, key_mask = ctx.saved_tensors
        return (*attention_backward(dout, q, k, v, out, lse, key_mask=key_mask, **ctx.args), None, None, None, None)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: Optional[int] = 0, sinks: int = 0,
              scale: Optional[float] = None, key_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out`` of :func:`attention_forward`, differentiable in q, k and v."""
    return _Attention.apply(q, k, v, window, sinks, scale, key_mask)


# ---------------------------------------------------------------- distillation
def _distill(logits, teacher_logits, teacher_ids, labels, temperature, alpha):
    zc = _float_code("logits", logits)
    if logits.dim() < 1 or logits.shape[-1] == 0:
        _fail(f"logits must be [..., vocab], got {tuple(logits.shape)}")
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    if teacher_logits.shape != teacher_ids.shape or teacher_ids.shape[:-1] != lead:
        _fail(f"teacher logits and ids must be {(*lead, 'k')}, got {tuple(teacher_logits.shape)} and {tuple(teacher_ids.shape)}")
    if labels is not None and labels.shape != lead:
        _fail(f"labels must be {tuple(lead)}, got {tuple(labels.shape)}")
    tc, ic = _float_code("teacher logits", teacher_logits), _index_code("teacher ids", teacher_ids)
    lc = 9 if labels is None else _index_code("labels", labels)
    _same_device(logits, teacher_logits=teacher_logits, teacher_ids=teacher_ids, labels=labels)
    z = _rows(logits, vocab)
    teacher_logits, teacher_ids = teacher_logits.contiguous(), teacher_ids.contiguous()
    labels = None if labels is None else labels.contiguous()
    head = (z.shape[0], vocab, zc, z.data_ptr(), z.stride(0), teacher_logits.data_ptr(), tc, teacher_ids.data_ptr(), ic,
            teacher_ids.shape[-1], _ptr(labels), lc, float(temperature), float(alpha))
    return z, (teacher_logits, teacher_ids, labels), head


def _row_weights(grad, z, lead):
    """A loss gradient per row as dense fp32."""
    if not isinstance(grad, torch.Tensor):
        return torch.full((z.shape[0],), float(grad), dtype=torch.float32, device=z.device)
    if grad.shape != lead or not grad.is_floating_point():
        _fail(f"grad must be {tuple(lead)} floating point values, got {tuple(grad.shape)} of {grad.dtype}")
    _same_device(z, grad=grad)
    return grad.to(torch.float32).contiguous()


def distill_loss_forward(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor, *,
                         labels: Optional[torch.Tensor] = None, temperature: float = 1.0, alpha: float = 1.0):
    """``(loss, stats)``: per row ``alpha * T^2 * KL(teacher || student)`` over the teacher's entries at
    temperature ``T``, plus ``(1 - alpha)`` times the cross-entropy of ``labels``.

    ``logits`` [..., vocab]; ``teacher_logits`` and ``teacher_ids`` [..., k] (k up to 1024): the teacher's
    distribution is the softmax of its entries.  An entry whose id lies outside the vocabulary (-1) is absent,
    a label outside it (-100) too; a row with neither has loss 0 and gradient 0.  ``loss`` is fp32 [...]."""
    z, keep, head = _distill(logits, teacher_logits, teacher_ids, labels, temperature, alpha)
    loss = torch.empty(logits.shape[:-1], dtype=torch.float32, device=z.device)
    stats = torch.empty((z.shape[0], 4), dtype=torch.float32, device=z.device)
    _call(z.device, lm_lib().stq_distill_forward, _DISTILL.pack(*head, loss.data_ptr(), stats.data_ptr(), 0, 0, 0))
    return loss, stats


def _grad_rows(logits, z, out):
    """Where the gradient goes: [..., vocab] and its rows."""
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    elif out.shape != logits.shape or out.dtype != logits.dtype:
        _fail(f"out must be {tuple(logits.shape)} of {logits.dtype}, got {tuple(out.shape)} of {out.dtype}")
    rows = out if out.dim() == 2 else out.view(-1, out.shape[-1])
    if rows.stride(1) != 1 and rows.shape[1] != 1:
        _fail("out must have dense rows")
    _same_device(z, out=out)
    return out, rows


def distill_loss_backward(grad, logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor, stats: torch.Tensor, *,
                          labels: Optional[torch.Tensor] = None, temperature: float = 1.0, alpha: float = 1.0,
                          out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient of the logits (their type) for ``grad``, the gradient of each row's loss.  ``out`` may be
    the logits themselves."""
    z, keep, head = _distill(logits, teacher_logits, teacher_ids, labels, temperature, alpha)
    if stats.dtype != torch.float32 or stats.shape != (z.shape[0], 4) or not stats.is_contiguous():
        _fail(f"stats must be the forward call's [{z.shape[0]}, 4]")
    w = _row_weights(grad, z, logits.shape[:-1])
    dz, rows = _grad_rows(logits, z, out)
    _same_device(z, stats=stats)
    _call(z.device, lm_lib().stq_distill_backward,
          _DISTILL.pack(*head, 0, stats.data_ptr(), w.data_ptr(), rows.data_ptr(), rows.stride(0)))
    if out is not None:
        _written(out)
    return dz


def distill_loss_and_grad(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor, *, grad,
                          labels: Optional[torch.Tensor] = None, temperature: float = 1.0, alpha: float = 1.0,
                          out: Optional[torch.Tensor] = None):
    """``(loss, dlogits)`` from one read of the logits: ``grad`` (a number, or one per row) is the gradient of
    each row's loss, 1 / rows for a mean.  ``out`` may be the logits themselves, which then hold the gradient."""
    z, keep, head = _distill(logits, teacher_logits, teacher_ids, labels, temperature, alpha)
    w = _row_weights(grad, z, logits.shape[:-1])
    loss = torch.empty(logits.shape[:-1], dtype=torch.float32, device=z.device)
    dz, rows = _grad_rows(logits, z, out)
    _call(z.device, lm_lib().stq_distill_forward,
          _DISTILL.pack(*head, loss.data_ptr(), 0, w.data_ptr(), rows.data_ptr(), rows.stride(0)))
    if out is not None:
        _written(out)
    return loss, dz


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_logits, teacher_ids, labels, temperature, alpha):
        loss, stats = distill_loss_forward(logits, teacher_logits, teacher_ids, labels=labels, temperature=temperature, alpha=alpha)
        ctx.save_for_backward(logits, teacher_logits, teacher_ids, labels, stats)
        ctx.args = dict(temperature=temperature, alpha=alpha)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        logits, teacher_logits, teacher_ids, labels, stats = ctx.saved_tensors
        dz = distill_loss_backward(grad, logits, teacher_logits, teacher_ids, stats, labels=labels, **ctx.args)
        return dz, None, None, None, None, None


def distill_loss(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor, *, labels: Optional[torch.Tensor] = None,
                 temperature: float = 1.0, alpha: float = 1.0) -> torch.Tensor:
    """``loss`` of :func:`distill_loss_forward` ([...], fp32), differentiable in ``logits``."""
    return _DistillLoss.apply(logits, teacher_logits, teacher_ids, labels, temperature, alpha)
