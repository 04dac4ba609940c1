"""Distillation calls that the other tests pass by, against the 64-bit oracle
(oracle/distill.py): temperatures whose log2(e)/T is an f32, lists without a
probability whose tokens repeat, teachers that require a gradient.  Tolerances
are test_distill_gpu.py's."""
import math

import numpy as np
import pytest
import torch

import pesti_distill as pd
from test_distill_gpu import _compare, _make

pytestmark = pytest.mark.gpu

NEG = float("-inf")
LOG2E = 1.4426950408889634


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("T", [1 / math.log(2), 2 / math.log(2), 0.5 / math.log(2), LOG2E / 1.25])
def test_temperatures_of_round_bases(dtype, tail, T):
    """The softmax to base 2 (4, the root of 2), over whole and ragged units, masked and not."""
    assert float(np.float32(LOG2E / T)) == LOG2E / T
    for V, pad in ((4096, 0), (3001, 1), (5, 0)):
        x, idx, val, lse = _make(4, V, 4, dtype, pad=pad, tail=tail, T=T)
        up = torch.tensor([1.0, -0.5, 2.0, 1.5]).cuda()
        _compare(x, idx, val, T, lse, None, dtype, up)
        unlisted = torch.ones(4, V, dtype=torch.bool).cuda().scatter_(1, idx.long(), False)
        x[1][unlisted[1] & (torch.arange(V).cuda() % 3 == 0)] = NEG
        x[2][unlisted[2]] = NEG
        x[3] = NEG
        _compare(x, idx, val, T, lse, None, dtype, up)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("weighted", [False, True])
def test_equal_tokens_without_probability(dtype, tail, weighted):
    """Rows padded as token 0 with -inf, wholly and behind real entries."""
    x, idx, val, lse = _make(5, 3001, 12, dtype, tail=tail)
    idx[0], val[0] = 0, NEG
    idx[1, 5:], val[1, 5:] = 0, NEG
    idx[2, 3], val[2] = idx[2, 9], NEG
    idx[3, :6], val[3] = -1, NEG
    idx[3, 6:] = 2999
    weight = torch.tensor([0.5, 1.0, 2.0, 0.25, 0.0]).cuda() if weighted else None
    _, grad = _compare(x, idx, val, 1.0, lse, weight, dtype)
    assert torch.isfinite(grad).all()
    if not tail:
        assert not grad[0].any() and not grad[2].any() and not grad[3].any()


def test_the_teacher_is_a_constant():
    """Values, weights and log sums that require a gradient get none, whether or not the logits do."""
    x, idx, val, lse = _make(6, 2000, 7, "f32", tail=True)
    w = torch.linspace(0.5, 1.0, 6).cuda()
    want = pd.distill_topk(x, idx, val, 1.0, lse, w)
    leaf = x.clone().requires_grad_()
    for t in (val, lse, w):
        t.requires_grad_()
    loss = pd.distill_topk(x, idx, val, 1.0, lse, w)
    assert torch.equal(loss, want) and not loss.requires_grad
    (loss.sum() + 3.0 * val.sum() + 2.0 * lse.sum() + w.sum()).backward()
    assert (val.grad == 3.0).all() and (lse.grad == 2.0).all() and (w.grad == 1.0).all()
    pd.distill_topk(leaf, idx, val, 1.0, lse, w).sum().backward()
    assert (val.grad == 3.0).all() and (lse.grad == 2.0).all() and (w.grad == 1.0).all()
    _, unit = pd.distill_topk_grad(x, idx, val.detach(), 1.0, lse.detach(), w.detach())
    assert torch.allclose(leaf.grad, unit, rtol=4 * 2.0 ** -24, atol=1e-12)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("T", [0.7, LOG2E / (1 + 2.0 ** -23 - 2.0 ** -40)])
@pytest.mark.parametrize("largest", [1.0e9, 7.0e8, 5.2e8, 3.0e8])
def test_logits_of_hundreds_of_millions(dtype, tail, T, largest):
    """Below the magnitude where only a row's largest logit counts, and just above it, at temperatures whose
    log2(e)/T lies nearly an f32 step above an f32."""
    m = largest * T / LOG2E
    x, idx, val, lse = _make(6, 2500, 6, dtype, tail=tail, T=T)
    x = x.contiguous()
    x[0] = m
    x[1] = -m
    x[2, ::2] = m        # half of them; the others, of order 1, have no probability
    x[3] = -m
    x[3, ::3] = -3.0 * m
    x[4, idx[4].long()] = m
    x[5] = m
    x[5, 7] = -m
    up = torch.linspace(0.5, 2.0, 6).cuda()
    _, grad = _compare(x, idx, val, T, lse, None, dtype, up)
    assert torch.isfinite(grad).all()
