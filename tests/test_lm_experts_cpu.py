"""Routing, expert products and clipping without a GPU: the packed structs have the header's layout, and bad arguments are
reported before any device work (the pointers below are never dereferenced)."""
import ctypes
import os
import struct
import types

import pytest
import torch

import stquant_lm as lm
from mdq_hip import _capi
from test_lm_cpu import INVALID, P, ROOT, err, fields


@pytest.mark.parametrize("name,packed", [("stq_route", lm._ROUTE), ("stq_expert_plan", lm._PLAN), ("stq_expert_product", lm._PRODUCT),
                                         ("stq_expert_combine", lm._COMBINE), ("stq_clip", lm._CLIP), ("stq_grad", struct.Struct("@QQqq"))])
def test_packed_structs_follow_the_header(name, packed):
    import re
    fmt = packed.format.replace("@", "").replace(" ", "").replace("Q", "q")
    flat = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([qd])", fmt))
    assert flat == fields(name) and packed.size == 8 * len(flat)


ROUTE = dict(n=4, e=8, k=2, dt=0, renorm=0, z=P, zs=8, w=P, ids=P, load=P, dw=P, dl=P, dz=P, dzs=8, ws=P, wsn=1 << 20)


def route(backward=False, **kw):
    L = _capi.lm_lib()
    return (L.stq_route_backward if backward else L.stq_route_forward)(lm._ROUTE.pack(*(ROUTE | kw).values()), None)


@pytest.mark.parametrize("backward,kw,msg", [
    (False, dict(dt=9), "logits must be Float, BFloat16 or Half, got Long"),
    (False, dict(e=0), "experts must be 1 to 512, got 0"),
    (False, dict(e=513), "experts must be 1 to 512, got 513"),
    (False, dict(k=0), "k must be 1 to 8, got 0"),
    (False, dict(k=9), "k must be 1 to 8, got 9"),
    (False, dict(e=512, k=65), "k must be 1 to 64, got 65"),
    (False, dict(n=-1), "n must be 0 to"),
    (False, dict(n=(1 << 29) + 1), "n must be 0 to 536870912"),
    (False, dict(renorm=2), "renormalize must be 0 or 1"),
    (False, dict(z=0), "logits: null data pointer"),
    (False, dict(z=P + 2), "logits must be aligned to 4 bytes"),
    (False, dict(zs=-1), "rows of logits: the stride must be >= 0"),
    (False, dict(w=0), "weights: null data pointer"),
    (False, dict(ids=P + 1), "ids must be aligned to 4 bytes"),
    (False, dict(load=P + 1), "load must be aligned to 4 bytes"),
    (False, dict(n=100, ws=0), "workspace: null data pointer"),
    (False, dict(n=100, wsn=100), "workspace needs 128 bytes, got 100"),
    (True, dict(dz=0), "dlogits: null data pointer"),
    (True, dict(dzs=7), "rows of dlogits must not overlap"),
    (True, dict(dw=P + 2), "dweights must be aligned to 4 bytes"),
])
def test_route_refusals(backward, kw, msg):
    assert route(backward, **kw) == INVALID and msg in err()


PLAN = dict(ids=P, idt=7, slots=10, e=4, rows=P, places=P, off=P, ws=0, wsn=0)


def plan(**kw):
    return _capi.lm_lib().stq_expert_plan_sort(lm._PLAN.pack(*(PLAN | kw).values()), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(idt=0), "ids must be Long or Int, got Float"),
    (dict(slots=(1 << 30) + 1), "slots must be 0 to 1073741824"),
    (dict(e=513), "experts must be 1 to 512"),
    (dict(off=0), "offsets: null data pointer"),
    (dict(ids=0), "ids: null data pointer"),
    (dict(rows=P + 2), "rows must be aligned to 4 bytes"),
    (dict(places=0), "places: null data pointer"),
    (dict(slots=100000), "workspace: null data pointer"),
    (dict(slots=100000, ws=P, wsn=16), "workspace needs 980 bytes, got 16"),
])
def test_plan_refusals(kw, msg):
    assert plan(**kw) == INVALID and msg in err()


PRODUCT = dict(dt=1, slots=12, e=4, din=16, dout=24, k=2, tokens=6, x=P, xs=16, w=P, wes=384, wrs=16, rows=P, places=P, off=P, y=P, dy=P, dys=24,
               dx=P, dw=P, dwdt=0, ws=P, wsn=1 << 20)


def product(backward=False, **kw):
    L = _capi.lm_lib()
    return (L.stq_expert_product_backward if backward else L.stq_expert_product_forward)(lm._PRODUCT.pack(*(PRODUCT | kw).values()), None)


@pytest.mark.parametrize("backward,kw,msg", [
    (False, dict(dt=0), "x and weight must be BFloat16 or Half, got Float"),
    (False, dict(e=0), "experts must be 1 to 512"),
    (False, dict(din=0), "in must be 8 to"),
    (False, dict(dout=(1 << 20) + 8), "out must be 8 to 1048576"),
    (False, dict(din=20), "in and out must be multiples of 8"),
    (False, dict(k=65), "k must be 0 to 64"),
    (False, dict(k=3), "slots (12) must be tokens (6) times k (3)"),
    (False, dict(tokens=1 << 62), "tokens must be 0 to"),
    (False, dict(slots=1 << 30, k=0, dout=1 << 20), "tiles of rows must be 0 to"),
    (False, dict(e=512, din=1 << 20, dout=1 << 20), "tiles of weights must be 0 to"),
    (False, dict(off=0), "offsets: null data pointer"),
    (False, dict(rows=0), "rows: null data pointer"),
    (False, dict(places=P + 2), "places must be aligned to 4 bytes"),
    (False, dict(x=P + 8), "x must be aligned to 16 bytes"),
    (False, dict(xs=20), "x: strides must be multiples of 8 elements"),
    (False, dict(w=P + 2), "weight must be aligned to 16 bytes"),
    (False, dict(wrs=-16), "weight: strides must be multiples of 8 elements"),
    (False, dict(wes=4), "weight: strides must be multiples of 8 elements"),
    (False, dict(y=0), "y: null data pointer"),
    (True, dict(dy=0), "dy: null data pointer"),
    (True, dict(dys=4), "dy: strides must be multiples of 8 elements"),
    (True, dict(dx=P + 4), "dx must be aligned to 16 bytes"),
    (True, dict(dwdt=2), "dweight must be Float or the type of x, got Half"),
    (True, dict(dw=P + 8), "dweight must be aligned to 16 bytes"),
    (True, dict(wsn=64), "workspace needs"),
    (True, dict(ws=P + 8), "workspace must be aligned to 16 bytes"),
])
def test_product_refusals(backward, kw, msg):
    assert product(backward, **kw) == INVALID and msg in err()


COMBINE = dict(n=6, k=2, e=4, dim=10, dt=0, y=P, ys=10, w=P, places=P, off=P, out=P, do=P, dos=10, dy=P, dw=P)


def combine(backward=False, **kw):
    L = _capi.lm_lib()
    return (L.stq_expert_combine_backward if backward else L.stq_expert_combine_forward)(lm._COMBINE.pack(*(COMBINE | kw).values()), None)


@pytest.mark.parametrize("backward,kw,msg", [
    (False, dict(dt=7), "y must be Float, BFloat16 or Half, got Int"),
    (False, dict(k=65), "k must be 1 to 64"),
    (False, dict(e=0), "experts must be 1 to 512"),
    (False, dict(n=1 << 30), "n must be 0 to"),
    (False, dict(dim=0), "dim must be 1 to"),
    (False, dict(w=P + 1), "weights must be aligned to 4 bytes"),
    (False, dict(places=0), "places: null data pointer"),
    (False, dict(off=0), "offsets: null data pointer"),
    (False, dict(y=0), "y: null data pointer"),
    (False, dict(ys=-1), "y_stride must be >= 0"),
    (False, dict(out=P + 2), "out must be aligned to 4 bytes"),
    (True, dict(do=0), "dout: null data pointer"),
    (True, dict(dos=-1), "dout_stride must be >= 0"),
    (True, dict(dy=0), "dy: null data pointer"),
    (True, dict(dw=P + 2), "dweights must be aligned to 4 bytes"),
])
def test_combine_refusals(backward, kw, msg):
    assert combine(backward, **kw) == INVALID and msg in err()


def clip(grads, max_norm=1.0, given=0, norm=P, ws=P, wsn=1 << 20, only_norm=False, count=None, null=False):
    flat = [v for g in grads for v in g]
    buf = ctypes.create_string_buffer(struct.pack(f"@{len(flat)}q", *flat), max(8 * len(flat), 1))
    L = _capi.lm_lib()
    fn = L.stq_grad_norm if only_norm else L.stq_clip_grads
    return fn(lm._CLIP.pack(0 if null else ctypes.addressof(buf), len(grads) if count is None else count, max_norm, given, norm, ws, wsn), None)


A, B = 0x100000, 0x200000
OVERLAP = "gradients that are written must not overlap others"


@pytest.mark.parametrize("grads,kw,msg", [
    ([(A, A, 10, 9)], {}, "gradients must be Float, BFloat16 or Half, got Long"),
    ([(A, A, -1, 0)], {}, "elements of a gradient must be 0 to"),
    ([(0, A, 10, 0)], {}, "grad: null data pointer"),
    ([(A + 2, A + 2, 10, 0)], {}, "grad must be aligned to 4 bytes"),
    ([(A, 0, 10, 0)], {}, "out: null data pointer"),
    ([(A, B + 1, 10, 1)], {}, "out must be aligned to 2 bytes"),
    ([(A, A, 10, 0)], dict(max_norm=-1.0), "max_norm must be >= 0"),
    ([(A, A, 10, 0)], dict(max_norm=float("nan")), "max_norm must be >= 0"),
    ([(A, A, 10, 0)], dict(norm=0), "norm: null data pointer"),
    ([(A, A, 10, 0)], dict(given=P + 2), "given norm must be aligned to 4 bytes"),
    ([(A, A, 10, 0)], dict(wsn=8), "workspace needs 16392 bytes, got 8"),
    ([(A, A, 10, 0)], dict(ws=P + 8), "workspace must be aligned to 16 bytes"),
    ([(A, A, 10, 0)], dict(null=True), "grads: null data pointer"),
    ([(A, A, 10, 0)], dict(count=-1), "count must be 0 to"),
    ([(A, A, 10, 0)], dict(only_norm=True, norm=0), "norm: null data pointer"),
    ([(A, A, 10, 0), (A, A, 10, 0)], {}, OVERLAP),                       # one tensor twice
    ([(A, A, 10, 0), (A + 36, A + 36, 10, 0)], {}, OVERLAP),
    ([(A, B, 10, 0), (B + 4096, B + 8, 10, 0)], {}, OVERLAP),            # two outputs
    ([(A, A + 8, 10, 0)], {}, OVERLAP),                                  # an output inside its own gradient
    ([(A, B, 10, 0), (B + 36, B + 4096, 10, 0)], {}, OVERLAP),           # an output inside another gradient
    ([(A, A, 1000, 0), (A + 8, B, 1, 0), (A + 64, B + 64, 1, 0)], {}, OVERLAP),
    ([(A, A, 1000, 0)], dict(given=A + 400), OVERLAP),                   # a given norm inside a gradient that is written
])
def test_clip_refusals(grads, kw, msg):
    assert clip(grads, **kw) == INVALID and msg in err()


def test_empty_calls_are_no_ops():
    assert route(n=0, load=0, z=0, w=0, ids=0) == _capi.STQ_OK and route(True, n=0, z=0) == _capi.STQ_OK
    assert product(slots=0, tokens=0, x=0, y=0) == _capi.STQ_OK
    assert product(True, slots=0, tokens=0, x=0, dy=0, dw=0) == _capi.STQ_OK
    assert combine(n=0, y=0) == _capi.STQ_OK and combine(True, n=0) == _capi.STQ_OK


def test_limits_of_a_launch():
    """Workgroups of 256 threads along one dimension: fewer than 2^24 of them for every size that is accepted."""
    def tiles(slots, experts, din, dout):
        wide, narrow = (max(din, dout) + 127) // 128, (min(din, dout) + 127) // 128
        return (slots // 128 + experts + 1) * wide, experts * wide * narrow
    assert max(tiles(1 << 23, 512, 11008, 4096)) < 1 << 24
    assert product(slots=1 << 24, k=0, dout=11008, din=4096, x=0) == INVALID and "tiles of rows" in err()
    assert product(slots=1 << 23, k=0, dout=11008, din=4096, x=0) == INVALID and "x: null data pointer" in err()


def test_limits_go_by_what_a_pass_writes():
    """Tiles are counted of the rows that a pass writes: y is as wide as out, dx as in, and a call without dx has none.  Wide inputs of
    narrow results, and runs of 2^30 rows, are inside (refused further on, for a null pointer, so that nothing runs)."""
    L = _capi.lm_lib()
    wide = dict(slots=1 << 24, tokens=1 << 21, k=8, din=8192, dout=64, x=0)
    for backward, kw in ((False, wide), (False, wide | dict(slots=131072, tokens=2048, k=64, din=1 << 20, dout=8)), (False, wide | dict(slots=1 << 30, k=0, din=8)),
                         (True, wide | dict(dx=0)), (True, wide | dict(slots=1 << 30, k=0, din=64, dout=8192))):
        assert product(backward, **kw) == INVALID and "x: null data pointer" in err()
    for backward, kw in ((False, wide | dict(din=64, dout=8200)), (True, wide | dict(din=8200)), (True, wide | dict(din=8200, k=0))):
        assert product(backward, **kw) == INVALID and "tiles of rows must be 0 to 8388608, got 8519680" in err()
    need = lambda **kw: L.stq_expert_product_workspace(lm._PRODUCT.pack(*(PRODUCT | wide | kw).values()))  # noqa: E731
    assert need(dx=0, din=8200) == 0 and need(din=64, dout=8200) == (1 << 24) * 64 * 4
    assert need(din=8200) == -1 and "tiles of rows" in err()
    # counted in 32 bits: full tiles, one that is not full for each expert and the rows of none, and a step beyond the last
    assert (1 << 23) + (512 + 1) * (1 << 13) + 512 < 1 << 32


def test_python_refusals():
    f, i = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    h = f.bfloat16()
    p = lm.ExpertPlan(torch.zeros(8, dtype=torch.int32), i, torch.zeros(4, dtype=torch.int32))
    w = torch.zeros(3, 16, 8, dtype=torch.bfloat16)
    for call, msg in [
        (lambda: lm.route_forward(f.double(), 2), "logits must be float32, bfloat16 or float16"),
        (lambda: lm.route_forward(f[:, :0], 2), r"logits must be \[..., experts\]"),
        (lambda: lm.route_forward(f, 2), "tensors must be CUDA"),
        (lambda: lm.expert_plan(f, 3), "ids must be int64 or int32"),
        (lambda: lm.expert_plan(i, 3), "tensors must be CUDA"),
        (lambda: lm.expert_product_forward(h, w[0], p), r"weight must be \[experts, out, in\]"),
        (lambda: lm.expert_product_forward(f, w, p), "x and weight must both be bfloat16 or both float16"),
        (lambda: lm.expert_product_forward(h, w, p._replace(rows=p.rows.long())), "the plan's rows must be dense int32"),
        (lambda: lm.expert_product_forward(h, w, p._replace(rows=p.rows[:7])), "not a plan"),
        # no choice a token: its gradient would never be written
        (lambda: lm.expert_product_forward(h, w, lm.ExpertPlan(p.rows[:0], i[:, :0].contiguous(), p.offsets), gather=True), "not a plan"),
        (lambda: lm.expert_plan(i[:, :0], 3), r"ids must be \[..., k\] with k > 0"),
        (lambda: lm.expert_product_forward(h, w, p), "tensors must be CUDA"),
        (lambda: lm.expert_combine_forward(f.double(), None, p), "y must be float32, bfloat16 or float16"),
        (lambda: lm.expert_combine_forward(f, None, p), "tensors must be CUDA"),
        (lambda: lm.grad_norm([f]), "tensors must be CUDA"),
        (lambda: lm.grad_norm([]), "no gradients"),
        (lambda: lm.clip_grads([f], 1.0, out=[]), "out must be 1 tensors, got 0"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            call()


def test_gradients_that_are_none():
    """A parameter that took no part in the step has none: said so, not an AttributeError, and the README's example leaves it out."""
    f = torch.zeros(4, 8)
    for call in (lambda: lm.grad_norm([None]), lambda: lm.grad_norm([f, None]), lambda: lm.clip_grads([None, f], 1.0), lambda: lm.clip_grads([f], 1.0, out=[None])):
        with pytest.raises(RuntimeError, match="must be tensors, got None"):
            call()
    readme = open(os.path.join(ROOT, "README.md")).read()
    lines = [line.split("#")[0].split("=", 1)[1] for line in readme.splitlines() if "lm.clip_grads(" in line]
    model, seen = torch.nn.ParameterList([torch.zeros(3), torch.zeros(5)]), []
    model[1].grad = torch.ones(5)
    for line in lines:
        eval(line, {"model": model, "lm": types.SimpleNamespace(clip_grads=lambda grads, most: seen.append(list(grads)))})
    assert lines and all(len(s) == 1 and s[0] is model[1].grad for s in seen)


def test_dense():
    t = torch.zeros(4, 6, 5)
    assert lm._dense(t) and lm._dense(t.transpose(0, 2)) and lm._dense(t.permute(1, 2, 0)) and lm._dense(t[:, :, :1].squeeze(-1)[:1, :1])
    assert not lm._dense(t[:, :3]) and not lm._dense(t[..., ::2]) and not lm._dense(t[:1].expand(4, 6, 5))
    assert lm._dense(torch.zeros(0, 3)) and lm._dense(torch.zeros(()))
