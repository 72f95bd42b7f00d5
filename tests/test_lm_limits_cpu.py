"""Limits of the transformer operators' C ABI that follow from their kernels' index types, without a GPU (the pointers
are never dereferenced)."""
import pytest

import stquant_lm as lm
from mdq_hip import _capi
from test_lm_cpu import INVALID, embed_grad, err, norm


def embed_grad_workspace(**kw):
    a = dict(tokens=0x10000, tdt=9, n=4, vocab=10, dim=8, grad=0x10000, gdt=0, gs=8, dw=0x10000, dwdt=0, dws=8, padding=-1, acc=0, ws=0, wsn=0, scale=1.0) | kw
    return _capi.lm_lib().stq_embedding_grad_workspace(lm._EMBED_GRAD.pack(*a.values()))


@pytest.mark.parametrize("name,most", [("n", 1 << 30), ("vocab", 1 << 30)])
def test_embedding_gradient_counts_within_32_bits(name, most):
    """Its kernels step past the last token or row in 32 bits: from 2^31 less a grid's surplus on that overflowed, and the
    sorted list was read in front of the workspace."""
    for v in (most + 1, (1 << 31) - 1):
        assert embed_grad(**{name: v}, wsn=1 << 50) == INVALID and f"{name} must be" in err()
        assert embed_grad_workspace(**{name: v}) == -1
    assert embed_grad_workspace(**{name: most}) > 0
    if name == "n":
        assert embed_grad(n=most) == INVALID and "workspace needs" in err()


def last_index(n, threads=64, seg=16):
    """The largest list index that the sums and the join form for n tokens (embed_sum_kernel, embed_join_kernel): the
    grid is whole layers of 32768 workgroups of 4 chunks."""
    wgs = ((n + seg - 1) // seg + 3) // 4
    layers = (wgs + 32767) // 32768
    chunks = min(wgs, 32768) * layers * 4
    return (chunks - 1) * seg - 1 + threads + seg


def test_the_limit_is_what_the_grid_needs():
    assert last_index(1 << 30) < 1 << 31
    assert last_index((1 << 31) - 1) >= 1 << 31          # (what was accepted before)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("kw", [dict(pb=0x10000, dpb=0x10000), dict(qw=0x10000, qb=0x10000, dqw=0x10000, dqb=0x10000)])
def test_rms_norms_refuse_biases(backward, kw):
    """They were accepted and left out of the result."""
    kw = kw if backward else {k: v for k, v in kw.items() if k[0] != "d"}
    assert norm(backward, **kw) == INVALID and "biases need layer norms" in err()


def test_a_gate_of_several_groups_without_rows():
    """No rows divide into any number of groups; what cannot be (rows and no group, a grid of sums beyond 65535) is refused."""
    assert norm(False, n=0, gate=0x10000, groups=5, x=0, block=0, r=0, h=0, stats=0) == _capi.STQ_OK
    for kw, msg in [(dict(gate=0x10000, groups=0), "gate rows must be 1 to 4"), (dict(n=0, gate=0x10000, groups=0), "gate rows must be 1 to"),
                    (dict(n=0, gate=0x10000, groups=1 << 31), "gate rows must be 1 to")]:
        assert norm(False, **kw) == INVALID and msg in err()
