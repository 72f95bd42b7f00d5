"""The transformer operators' C ABI and refusals, without a GPU: every symbol that include/stquant_lm.h declares is
exported, the packed argument structs have the header's layout, and bad arguments are reported before any device work
(the pointers below are never dereferenced)."""
import os
import re

import pytest
import torch

import mdq_hip
import stquant_lm as lm
from mdq_hip import _capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = open(os.path.join(ROOT, "include", "stquant_lm.h")).read()
P, INVALID = 0x10000, _capi.STQ_ERR_INVALID


def err():
    return mdq_hip.lib().stq_last_error().decode()


def test_exports_every_declared_symbol():
    names = set(re.findall(r"^\s*(?:int|int64_t)\s+(stq_\w+)\s*\(", HEADER, re.M))
    assert names == set(_capi.LM_SYMBOLS)
    L = _capi.lm_lib()
    assert all(hasattr(L, n) for n in names)
    assert L.stq_lm_abi_version() == _capi.LM_ABI_VERSION == int(re.search(r"STQ_LM_ABI_VERSION (\d+)", HEADER)[1])


def fields(name):
    """A struct's fields in order: 'd' for double, 'q' for everything else (all are 8 bytes)."""
    body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), HEADER, re.S)[1], flags=re.S)
    out = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        kind = decl.split()[0] if not decl.startswith("const") else "pointer"
        names = [n for n in decl.split(",")]
        width = 4 if kind == "stq_tensor4" else 1
        out += ["d" if kind == "double" else "q"] * width * len(names)
    return "".join(out)


@pytest.mark.parametrize("name,packed", [("stq_embedding", lm._EMBED), ("stq_embedding_grad", lm._EMBED_GRAD), ("stq_norm_residual", lm._NORM),
                                         ("stq_attention", lm._ATTN), ("stq_distill", lm._DISTILL)])
def test_packed_structs_follow_the_header(name, packed):
    fmt = packed.format.replace("@", "").replace(" ", "").replace("Q", "q")
    flat = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([qd])", fmt))
    assert flat == fields(name) and packed.size == 8 * len(flat)


def embed(**kw):
    a = dict(tokens=P, tdt=9, n=4, vocab=10, dim=8, weight=P, wdt=0, ws=8, out=P, odt=0, scale=1.0) | kw
    return _capi.lm_lib().stq_embedding_forward(lm._EMBED.pack(*a.values()), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(tdt=5), "tokens must be Long or Int, got Short"),
    (dict(wdt=4), "weight must be Float, BFloat16 or Half, got Char"),
    (dict(odt=9), "out must be Float, BFloat16 or Half, got Long"),
    (dict(n=-1), "n must be 0 to"),
    (dict(vocab=0), "vocab must be 1 to"),
    (dict(dim=0), "dim must be 1 to"),
    (dict(tokens=0), "tokens: null data pointer"),
    (dict(tokens=P + 4), "tokens must be aligned to 8 bytes"),
    (dict(weight=0), "weight: null data pointer"),
    (dict(weight=P + 2), "weight must be aligned to 4 bytes"),
    (dict(out=P + 1, odt=1), "out must be aligned to 2 bytes"),
    (dict(scale=float("nan")), "scale must be finite"),
    (dict(ws=-8), "weight_stride must be >= 0"),
])
def test_embedding_refusals(kw, msg):
    assert embed(**kw) == INVALID and msg in err()


def embed_grad(**kw):
    a = dict(tokens=P, tdt=9, n=4, vocab=10, dim=8, grad=P, gdt=0, gs=8, dw=P, dwdt=0, dws=8, padding=-1, acc=0, ws=P, wsn=1 << 20, scale=1.0) | kw
    return _capi.lm_lib().stq_embedding_backward(lm._EMBED_GRAD.pack(*a.values()), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(gdt=7), "grad must be Float, BFloat16 or Half, got Int"),
    (dict(dws=7), "rows of dweight must not overlap"),
    (dict(ws=0), "workspace: null data pointer"),
    (dict(wsn=8), "workspace needs"),
    (dict(grad=0), "grad: null data pointer"),
])
def test_embedding_gradient_refusals(kw, msg):
    assert embed_grad(**kw) == INVALID and msg in err()


NORM = dict(n=4, dim=16, dt=1, wdt=1, x=P, block=P, xs=16, bs=16, pw=P, pb=0, qw=0, qb=0, gate=0, groups=1, layer=0, rs=1.0, eps=1e-5, stats=P,
            r=P, h=P, dr=P, dh=P, drs=16, dhs=16, dx=P, dblock=P, dpw=P, dpb=0, dqw=0, dqb=0, dgate=0, ws=P, wsn=1 << 24)


def norm(backward, **kw):
    L = _capi.lm_lib()
    return (L.stq_norm_residual_backward if backward else L.stq_norm_residual_forward)(lm._NORM.pack(*(NORM | kw).values()), None)


@pytest.mark.parametrize("backward,kw,msg", [
    (False, dict(dt=9), "x must be Float, BFloat16 or Half, got Long"),
    (False, dict(wdt=2), "weights must be Float or the type of x, got Half"),
    (False, dict(dim=7), "dim must be 8 to 8192, got 7"),
    (False, dict(dim=8193), "dim must be 8 to 8192, got 8193"),
    (False, dict(pw=0), "pre_weight: null data pointer"),
    (False, dict(qb=P), "post_bias needs post_weight"),
    (False, dict(gate=P, groups=3), "gate rows (3) must divide the rows (4)"),
    (False, dict(gate=P, groups=5), "gate rows must be 1 to 4"),
    (False, dict(layer=2), "layer must be 0 or 1"),
    (False, dict(eps=-1.0), "eps must be finite and >= 0"),
    (False, dict(rs=float("inf")), "residual_scale must be finite"),
    (False, dict(x=P + 1), "x must be aligned to 2 bytes"),
    (False, dict(r=0), "r: null data pointer"),
    (True, dict(dpw=0), "the gradient of pre_weight goes with it"),
    (True, dict(dgate=P), "the gradient of gate goes with it"),
    (True, dict(dh=0), "dh: null data pointer"),
    (True, dict(wsn=16), "workspace needs"),
    (True, dict(ws=P + 8), "workspace must be aligned to 16 bytes"),
])
def test_norm_refusals(backward, kw, msg):
    assert norm(backward, **kw) == INVALID and msg in err()


ATTN_HEAD = dict(dt=1, b=2, h=4, hk=2, t=8, s=8, d=64, window=0, sinks=0, scale=0.125)


def attention(backward=False, t4=None, **kw):
    a = ATTN_HEAD | {k: v for k, v in kw.items() if k in ATTN_HEAD}
    four = {n: (P, 2048, 512, 64) for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv")} | (t4 or {})
    flat = lambda *names: [x for n in names for x in four[n]]  # noqa: E731
    packed = lm._ATTN.pack(*a.values(), *flat("q", "k", "v", "out"), 0, 0, kw.get("lse", P), *flat("dout", "dq", "dk", "dv"), kw.get("ws", P), kw.get("wsn", 1 << 20))
    L = _capi.lm_lib()
    return (L.stq_attention_backward if backward else L.stq_attention_forward)(packed, None)


@pytest.mark.parametrize("backward,kw,msg", [
    (False, dict(dt=0), "q, k and v must be BFloat16 or Half, got Float"),
    (False, dict(h=5), "heads (5) must be a multiple of key_heads (2)"),
    (False, dict(t=9), "rows must be 0 to 8, got 9"),
    (False, dict(d=136), "dim must be 8 to 128"),
    (False, dict(d=60), "dim must be a multiple of 8, got 60"),
    (False, dict(window=-1), "window and sinks must be >= 0"),
    (False, dict(scale=0.0), "scale must be finite and > 0"),
    (False, dict(b=40000), "batch * key_heads must be 0 to 65535"),
    (False, dict(t4={"q": (P + 8, 2048, 512, 64)}), "q must be aligned to 16 bytes"),
    (False, dict(t4={"v": (P, 2048, 512, 60)}), "v: strides must be multiples of 8 elements"),
    (False, dict(t4={"out": (0, 2048, 512, 64)}), "out: null data pointer"),
    (False, dict(lse=0), "lse: null data pointer"),
    (True, dict(t4={"dk": (P, 2048, 511, 64)}), "dk: strides must be multiples of 8 elements"),
    (True, dict(t4={"dout": (0, 0, 0, 0)}), "dout: null data pointer"),
    (True, dict(wsn=100), "workspace needs 256 bytes, got 100"),
])
def test_attention_refusals(backward, kw, msg):
    assert attention(backward, **kw) == INVALID and msg in err()


DISTILL = dict(n=4, v=100, dt=1, z=P, zs=100, t=P, tdt=0, ids=P, idt=9, k=5, lab=0, ldt=9, temp=1.0, alpha=0.5, loss=P, stats=P, drow=P, dz=0, dzs=0)


@pytest.mark.parametrize("backward,kw,msg", [
    (False, dict(scale=1e-40), "scale must be finite and > 0"),        # a float of 0
    (False, dict(scale=1e39), "scale must be finite and > 0"),         # an infinite float
    (False, dict(t4=dict(k=(P, 2048, 512, (1 << 22) + 8))), "k: row_stride must be 0 to 2^22"),
    (False, dict(t4=dict(v=(P, 2048, -8, 64))), "v: row_stride must be 0 to 2^22, head_stride >= 0"),
    (False, dict(t4=dict(q=(P, 2048, (1 << 28) + 8, 64))), "q and dout: the heads of a key head must lie within 2^29"),
    (True, dict(t4=dict(dout=(P, 2048, (1 << 28) + 8, 64))), "q and dout: the heads of a key head must lie within 2^29"),
    (False, dict(b=40000), "batch * key_heads must be 0 to 65535"),
    (False, dict(t=8, s=(1 << 22) + 1), "keys must be 0 to"),
    (False, dict(t=(1 << 21) + 1, s=1 << 22), "rows * heads / key_heads must be 0 to"),
])
def test_attention_limits(backward, kw, msg):
    assert attention(backward, **kw) == INVALID and msg in err()


@pytest.mark.parametrize("temperature", [1e-30, 1e-16, 1e16, 1e39])
def test_distill_temperatures_outside_the_floats(temperature):
    assert distill(temp=temperature) == INVALID and "temperature must be finite and > 0" in err()


def distill(backward=False, **kw):
    L = _capi.lm_lib()
    return (L.stq_distill_backward if backward else L.stq_distill_forward)(lm._DISTILL.pack(*(DISTILL | kw).values()), None)


@pytest.mark.parametrize("backward,kw,msg", [
    (False, dict(dt=7), "logits must be Float, BFloat16 or Half, got Int"),
    (False, dict(tdt=9), "teacher logits must be Float, BFloat16 or Half, got Long"),
    (False, dict(idt=0), "teacher ids must be Long or Int, got Float"),
    (False, dict(lab=P, ldt=5), "labels must be Long or Int, got Short"),
    (False, dict(v=0), "vocab must be 1 to"),
    (False, dict(k=1025), "teacher entries must be 0 to 1024, got 1025"),
    (False, dict(temp=0.0), "temperature must be finite and > 0"),
    (False, dict(alpha=1.5), "alpha must be 0 to 1"),
    (False, dict(z=P + 1), "logits must be aligned to 2 bytes"),
    (False, dict(stats=0), "stats: null data pointer"),
    (False, dict(dz=P, dzs=99), "rows of logits must not overlap"),
    (False, dict(dz=P + 64, dzs=100), "dlogits must be the logits or lie apart from them"),
    (False, dict(dz=P + 4096, dzs=100, drow=0), "drow: null data pointer"),
    (True, dict(), "dlogits: null data pointer"),
])
def test_distill_refusals(backward, kw, msg):
    assert distill(backward, **kw) == INVALID and msg in err()


def test_empty_calls_are_no_ops():
    assert embed(n=0, tokens=0, weight=0, out=0) == _capi.STQ_OK
    assert norm(False, n=0, x=0, block=0, r=0, h=0, stats=0) == _capi.STQ_OK
    assert attention(b=0) == _capi.STQ_OK and attention(t=0) == _capi.STQ_OK
    assert distill(n=0, z=0) == _capi.STQ_OK


def test_null_arguments_are_refused():
    L = _capi.lm_lib()
    for name in _capi.LM_SYMBOLS:
        if name.endswith("version"):
            continue
        rc = getattr(L, name)(None) if name.endswith("_workspace") else getattr(L, name)(None, None)
        assert rc in (INVALID, -1) and "null arguments" in err(), name


def test_python_refusals():
    f, i = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    for call, msg in [
        (lambda: lm.embedding_forward(i.float(), f), "tokens must be int64 or int32"),
        (lambda: lm.embedding_forward(i, f.double()), "weight must be float32, bfloat16 or float16"),
        (lambda: lm.embedding_forward(i, f[0]), r"weight must be \[vocab, dim\]"),
        (lambda: lm.embedding_forward(i, f), "tensors must be CUDA"),
        (lambda: lm.embedding_backward(f[:3], i, 9), "grad must be"),
        (lambda: lm.norm_residual_forward(f, f[:2], f[0]), "x and block must have one shape"),
        (lambda: lm.norm_residual_forward(f, f.bfloat16(), f[0]), "block must be torch.float32"),
        (lambda: lm.norm_residual_forward(f, f, f[0]), "tensors must be CUDA"),
        (lambda: lm.attention_forward(f, f, f), "q, k, v must be"),
        (lambda: lm.attention_forward(f.view(1, 1, 4, 8), f.view(1, 1, 4, 8), f.view(1, 1, 4, 8)), "all be bfloat16 or all float16"),
        (lambda: lm.attention_forward(*(torch.zeros(1, 1, n, 8, dtype=torch.bfloat16) for n in (5, 4, 4))), "5 positions cannot be the last of 4 keys"),
        (lambda: lm.attention_forward(*(torch.zeros(1, 1, 4, 8, dtype=torch.bfloat16) for _ in range(3))), "tensors must be CUDA"),
        (lambda: lm.distill_loss_forward(f, f, i), "teacher logits and ids must be"),
        (lambda: lm.distill_loss_forward(f, f[:, :2], torch.zeros(4, 2, dtype=torch.int64)), "tensors must be CUDA"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            call()
    with pytest.raises(ValueError, match="kind must be 'rms' or 'layer'"):
        lm.norm_residual_forward(f, f, f[0], kind="batch")
