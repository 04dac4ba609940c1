"""Top-logit distillation on the GPU against the 64-bit oracle
(oracle/distill.py): losses, gradients from both entry points, autograd.

Tolerances.  A row's sum S of 2^t is off by at most: the hardware's 2^t,
2^-22.5; two roundings of t, ln 2 * 2 * 2^-24 * E[|t|] with E[|t|] <= log2(V) + 2
<= 20, so 1.7e-6; up to 24 f32 additions, 1.5e-6.  Together 3.4e-6, which is
also the error of every log p and, in the tail's p_t, counts twice:
  |loss - exact| <= 7e-6 w T^2 (Q + q_t) + half an f32 step.
A gradient entry outside the list is A 2^t: relative to its two parts
(Q + q_t) p and q_t/p_t p, S's error, 2^t's own with |t| <= 150 (1.3e-5) and two
f32 roundings: 2e-5; inside the list p is in 64 bits but for S.  Then half a
step of the type, or of its smallest subnormal."""
import numpy as np
import pytest
import torch
from torch.utils.checkpoint import checkpoint

import distill as OD
import pesti_beam as pb
import pesti_distill as pd

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TINY = {"f32": 2.0 ** -120, "bf16": 2.0 ** -120, "f16": 2.0 ** -25}


def _make(N, V, k, dtype, val="f32", pad=0, seed=0, tail=False, T=1.0):
    g = torch.Generator().manual_seed(seed * 104729 + N * 31 + V * 7 + k)
    base = torch.randn(N, V, generator=g) * 3
    kk = min(k, V)
    v, i = torch.topk(base, kk, dim=1)
    idx = torch.full((N, k), -1, dtype=torch.int32)
    vals = torch.zeros(N, k)
    idx[:, :kk], vals[:, :kk] = i.to(torch.int32), v
    x = torch.zeros(N, V + pad, dtype=DT[dtype])
    x[:, :V] = (0.8 * base + torch.randn(N, V, generator=g)).to(DT[dtype])
    lse = torch.logsumexp(base / T, 1).cuda() if tail else None
    return x.cuda()[:, :V], idx.cuda(), vals.to(DT[val]).cuda(), lse


def _np(t):
    return None if t is None else t.detach().float().cpu().numpy()


def _compare(x, idx, val, T, lse, weight, dtype, up=None):
    """Losses and gradients of the fused call and of forward + backward."""
    N, V = x.shape
    loss, grad, p, total, ratio = OD.batch(_np(x), idx.cpu().numpy(), _np(val), T, _np(lse), _np(weight))
    w = np.ones(N) if weight is None else np.abs(_np(weight).astype(np.float64))
    u = np.ones(N) if up is None else _np(up).astype(np.float64)
    got_l, got_g = pd.distill_topk_grad(x, idx, val, temperature=T, teacher_lse=lse, weight=weight)
    leaf = x.detach().clone() if x.is_contiguous() else x.detach()
    leaf.requires_grad_()
    l2 = pd.distill_topk(leaf, idx, val, temperature=T, teacher_lse=lse, weight=weight)
    g2, = torch.autograd.grad(l2, leaf, torch.ones_like(l2) if up is None else up)
    assert torch.equal(torch.isnan(l2), torch.isnan(got_l))
    half = float(torch.finfo(DT[dtype]).eps) / 2
    for l, g, scale in ((got_l, got_g, np.ones(N)), (l2, g2, u)):
        l, g = _np(l).astype(np.float64), _np(g).astype(np.float64)
        fine = np.isfinite(loss)
        assert np.array_equal(np.isnan(l), np.isnan(loss))
        assert np.array_equal(l[np.isinf(loss)], loss[np.isinf(loss)])
        tol = 7e-6 * w * T * T * np.maximum(total, 1e-30) + np.abs(loss) * 2.0 ** -24
        assert np.all(np.abs(l[fine] - loss[fine]) <= tol[fine])
        want = grad * scale[:, None]
        assert np.array_equal(np.isnan(g), np.isnan(want))
        s = (w * np.abs(scale) * T)[:, None]
        tol = 2e-5 * s * p * (total + ratio)[:, None] + np.abs(want) * half * 1.001 + TINY[dtype]
        bad = ~np.isnan(want) & ~(np.abs(g - want) <= tol)
        assert not bad.any(), (np.argwhere(bad)[:4], g[bad][:4], want[bad][:4], tol[bad][:4])
    return got_l, got_g


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("N,V,k,pad,T", [
    (1, 1, 1, 0, 1.0), (2, 2, 1, 1, 0.7), (3, 7, 9, 0, 1.0), (1, 1000, 20, 0, 2.0), (5, 4099, 33, 1, 1.5),
    (4, 2048, 256, 0, 1.0), (9, 32001, 20, 0, 4.0), (2, 128256, 64, 8, 1.0), (40, 3000, 5, 3, 0.3),
])
def test_against_the_oracle(dtype, tail, N, V, k, pad, T):
    x, idx, val, lse = _make(N, V, k, dtype, pad=pad, tail=tail, T=T)
    weight = torch.linspace(0.0, 1.5, N).cuda() if N > 2 else None
    up = torch.linspace(-1.0, 2.0, N).cuda()
    _compare(x, idx, val, T, lse, weight, dtype, up)


@pytest.mark.parametrize("val", ["bf16", "f16"])
def test_teacher_types(val):
    x, idx, v, _ = _make(6, 5000, 40, "bf16", val=val)
    _compare(x, idx, v, 1.0, None, None, "bf16")


@pytest.mark.parametrize("N", [1, 3])
def test_long_rows(N):
    x, idx, val, lse = _make(N, 620_003, 16, "bf16", tail=True)
    _compare(x, idx, val, 1.0, lse, None, "bf16")
    x, idx, val, lse = _make(N, 300_001, 16, "f32")
    _compare(x, idx, val, 1.0, lse, None, "f32")


# large batches: many rows, many units, rows of weight 0 between others
@pytest.mark.parametrize("N,V,dtype,tail,pad", [
    (210, 128256, "bf16", True, 0), (400, 32001, "f32", False, 1), (13, 2_000_003, "f16", True, 0),
    (9000, 3001, "bf16", True, 1),
])
def test_large_calls(N, V, dtype, tail, pad):
    x, idx, val, lse = _make(N, V, 20, dtype, tail=tail, pad=pad)
    weight = torch.linspace(0.5, 1.5, N).cuda()
    weight[::7] = 0.0
    weight[1::50] = 0.0
    x[0] = float("nan")  # of weight 0: not read
    _compare(x, idx, val, 1.0, lse, weight, dtype)
    first = pd.distill_topk_grad(x, idx, val, teacher_lse=lse, weight=weight)
    for _ in range(3):
        again = pd.distill_topk_grad(x, idx, val, teacher_lse=lse, weight=weight)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    # in place, and nothing between the rows is written
    behind = x.as_strided((N - 1, 1), (V + pad, 1), V).clone() if pad else None
    loss, grad = pd.distill_topk_grad(x, idx, val, teacher_lse=lse, weight=weight, grad=x)
    assert torch.equal(loss, first[0]) and torch.equal(x, first[1])
    if pad:
        assert torch.equal(x.as_strided((N - 1, 1), (V + pad, 1), V), behind)


def test_large_calls_at_once_and_captured():
    """Two large calls on two streams at the same time, and in graphs replayed together."""
    a = [_make(220, 128256, 16, "bf16", tail=True, seed=s) for s in (1, 2)]
    want = [pd.distill_topk_grad(x, i, v, teacher_lse=l) for x, i, v, l in a]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        got = [pd.distill_topk_grad(x, i, v, teacher_lse=l, stream=s.cuda_stream)
               for (x, i, v, l), s in zip(a, streams)]
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
    graphs, outs = [], []
    for x, i, v, l in a:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(pd.distill_topk_grad(x, i, v, teacher_lse=l))
        graphs.append(g)
    for _ in range(4):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tail", [False, True])
def test_lists(dtype, tail):
    """Padding, tokens outside the vocabulary, tokens listed twice, empty lists,
    zero probabilities, lists in any order."""
    N, V, k = 8, 3001, 12
    x, idx, val, lse = _make(N, V, k, dtype, tail=tail)
    idx[0] = -1
    idx[1, 3:] = -1
    idx[2, 4] = V
    idx[2, 5] = 2**31 - 1
    idx[2, 6] = -2**31
    idx[3, 7] = idx[3, 2]
    idx[4] = idx[4, 0]
    val[5, 4:] = float("-inf")
    val[6] = float("-inf")
    idx[7] = idx[7].flip(0)
    val[7] = val[7].flip(0)
    if tail:
        # a token that stands for several entries must not raise the sum above 1
        lse[3] += 0.7
        lse[4] += 3.0
    _compare(x, idx, val, 1.0, lse, None, dtype)


def test_tail_of_nothing():
    """A list of the whole vocabulary, and one whose complement is masked."""
    x, idx, val, lse = _make(3, 40, 40, "f32", tail=True)
    _compare(x, idx, val, 1.0, lse, None, "f32")
    x, idx, val, lse = _make(3, 40, 8, "f32", tail=True)
    listed = torch.zeros(3, 40, dtype=torch.bool).cuda().scatter_(1, idx.long(), True)
    x = torch.where(listed, x, torch.full_like(x, float("-inf")))
    _compare(x, idx, val, 1.0, lse, None, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("T", [1.0, 1.5])
def test_masks_and_extreme_logits(dtype, tail, T):
    N, V, k = 13, 2500, 6
    x, idx, val, lse = _make(N, V, k, dtype, tail=tail, T=T)
    x = x.contiguous()
    low = torch.finfo(x.dtype).min
    unlisted = torch.ones(N, V, dtype=torch.bool).cuda().scatter_(1, idx.long(), False)
    x[0] = float("-inf")
    x[1][unlisted[1]] = float("-inf")
    x[2, idx[2, 0].long()] = float("-inf")   # a listed token without probability
    x[3] = low                               # a mask of the lowest value over everything
    x[4][unlisted[4]] = low
    x[5, 1::2] = low
    x[6, 77] = float("nan")
    x[7, 78] = float("inf")
    x[8, idx[8, 1].long()] = float("nan")
    x[9, idx[9, 1].long()] = float("inf")
    x[10] = 0.0
    x[11] = 60000.0
    x[12, 5] = 300.0
    if tail:
        # the tail's mass lies below what f32 holds of it: 64 bits on both sides
        x[12, idx[12, 0].long()] = 320.0
    _compare(x, idx, val, T, lse, None, dtype)


def test_nan_in_the_list():
    x, idx, val, lse = _make(4, 500, 6, "f32", tail=True)
    val[1, 2] = float("nan")
    val[2, 2] = float("nan")
    idx[2, 2] = -1  # padding: not looked at
    _compare(x, idx, val, 1.0, None, None, "f32")
    _compare(x, idx, val, 1.0, lse, None, "f32")


def test_rows_of_weight_zero_are_not_read():
    x, idx, val, _ = _make(4, 5000, 8, "bf16")
    x[1] = float("nan")
    x[3, 7] = float("inf")
    w = torch.tensor([1.0, 0.0, 2.0, 0.0]).cuda()
    loss, grad = pd.distill_topk_grad(x, idx, val, weight=w)
    assert torch.isfinite(loss).all() and torch.isfinite(grad).all()
    assert loss[1] == 0 and loss[3] == 0 and not grad[1].any() and not grad[3].any()
    leaf = x.clone().requires_grad_()
    pd.distill_topk(leaf, idx, val, weight=w).sum().backward()
    assert torch.equal(leaf.grad[1], torch.zeros_like(leaf.grad[1])) and torch.isfinite(leaf.grad).all()


@pytest.mark.parametrize("dtype,V", [("f32", 32000), ("bf16", 128256), ("bf16", 32001), ("f16", 700_001)])
def test_gradient_in_place(dtype, V):
    x, idx, val, lse = _make(5, V, 16, dtype, tail=True, pad=1)
    loss, grad = pd.distill_topk_grad(x, idx, val, teacher_lse=lse)
    keep_pad = x.as_strided((5, 1), (V + 1, 1), V).clone()
    l2, g2 = pd.distill_topk_grad(x, idx, val, teacher_lse=lse, grad=x)
    assert torch.equal(loss, l2) and torch.equal(grad, x)
    assert torch.equal(x.as_strided((5, 1), (V + 1, 1), V), keep_pad)  # nothing behind the rows is written
    assert g2.data_ptr() == x.data_ptr()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_outputs_of_another_alignment(dtype):
    """Logits and gradient rows that start at different places of a 16-byte line: every shift between them."""
    x, idx, val, _ = _make(4, 9100, 8, dtype, pad=0)
    _, want = pd.distill_topk_grad(x, idx, val)
    for shift in range(1, 9):
        buf = torch.full((4, 9117), 7.0, dtype=DT[dtype], device="cuda")
        pd.distill_topk_grad(x, idx, val, grad=buf[:, shift:shift + 9100])
        assert torch.equal(buf[:, shift:shift + 9100], want), shift
        assert (buf[:, :shift] == 7).all() and (buf[:, shift + 9100:] == 7).all()


def test_same_bits_every_time():
    x, idx, val, lse = _make(64, 32000, 64, "bf16", tail=True)
    first = pd.distill_topk_grad(x, idx, val, teacher_lse=lse)
    for _ in range(5):
        again = pd.distill_topk_grad(x, idx, val, teacher_lse=lse)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_gradient_against_differences():
    """Autograd's gradient against central differences of the oracle's loss
    (h = 1e-4: h^2/6 of third derivatives below 10) within the f32 tolerance."""
    x, idx, val, lse = _make(2, 30, 6, "f32", tail=True)
    leaf = x.clone().requires_grad_()
    pd.distill_topk(leaf, idx, val, temperature=1.3, teacher_lse=lse).sum().backward()
    g = _np(leaf.grad)
    h = 1e-4
    for n in range(2):
        for v in range(30):
            d = np.zeros(30)
            d[v] = h
            at = _np(x)[n].astype(np.float64)
            args = (idx.cpu().numpy()[n], _np(val)[n], 1.3, float(lse[n]))
            diff = (OD.row(at + d, *args)[0] - OD.row(at - d, *args)[0]) / (2 * h)
            assert abs(diff - g[n, v]) <= 2e-5 + 2e-8


@pytest.mark.parametrize("reduce", ["sum", "mean", "rows", "expanded"])
def test_upstream_gradients(reduce):
    x, idx, val, _ = _make(6, 3000, 10, "f32")
    _, unit = pd.distill_topk_grad(x, idx, val)
    leaf = x.clone().requires_grad_()
    loss = pd.distill_topk(leaf, idx, val)
    up = torch.ones(6).cuda()
    if reduce == "sum":
        loss.sum().backward()
    elif reduce == "mean":
        loss.mean().backward()
        up = up / 6
    elif reduce == "rows":
        up = torch.arange(6.0).cuda()
        loss.backward(up)
    else:
        loss.backward(torch.full((1,), 2.0).cuda().expand(6))
        up = up * 2
    # three f32 roundings apart
    assert torch.allclose(leaf.grad, unit * up[:, None], rtol=4 * 2.0 ** -24, atol=1e-12)


def test_autograd_through_a_head():
    """Gradients reach the weights before the logits, twice through the same
    graph, and no gradient is asked of the teacher."""
    g = torch.Generator().manual_seed(2)
    h = torch.randn(10, 64, generator=g).cuda().bfloat16()
    W = (torch.randn(64, 4001, generator=g) * 0.1).cuda().bfloat16().requires_grad_()
    _, idx, val, _ = _make(10, 4001, 16, "bf16")
    logits = h @ W
    loss = pd.distill_topk(logits, idx, val, temperature=2.0).mean()
    gW, = torch.autograd.grad(loss, W, retain_graph=True)
    again, = torch.autograd.grad(loss, W)
    _, dl = pd.distill_topk_grad(logits, idx, val, temperature=2.0, weight=torch.full((10,), 0.1).cuda())
    want = h.float().t() @ dl.float()
    assert torch.equal(gW, again)
    # bf16 gradients of the logits (2^-8 each, twice) and a bf16 product
    assert (gW.float() - want).norm() <= 3 * 2.0 ** -8 * want.norm()
    with torch.no_grad():
        assert not pd.distill_topk(logits, idx, val).requires_grad


def test_overwritten_logits_have_no_backward():
    x, idx, val, _ = _make(4, 500, 5, "f32")
    y = x.clone().requires_grad_()
    loss = pd.distill_topk(y, idx, val)
    pd.distill_topk_grad(y, idx, val, grad=y.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.sum().backward()


@pytest.mark.parametrize("tail", [False, True])
def test_saved_tensors_may_move(tail):
    # hooks hand other tensors to the backward call: copies whose rows are padded, the originals overwritten
    x, idx, val, lse = _make(5, 2051, 7, "bf16", pad=3, tail=tail)
    up = torch.rand(5, device="cuda")

    def padded(t):
        t = t.detach()
        room = t.new_zeros(t.shape[0], *[n + 5 for n in t.shape[1:]])
        view = room[tuple(slice(0, n) for n in t.shape)]
        return view.copy_(t)

    def gradient(hooks):
        y = x.clone().requires_grad_()
        i, v, l = idx.clone(), val.clone(), lse.clone() if tail else None
        if not hooks:
            pd.distill_topk(y, i, v, 2.0, l).backward(up)
            return y.grad
        with torch.autograd.graph.saved_tensors_hooks(padded, lambda t: t):
            loss = pd.distill_topk(y, i, v, 2.0, l)
        with torch.no_grad():
            y.zero_(), v.zero_(), i.zero_()
            if tail:
                l.zero_()
        loss.backward(up)
        return y.grad

    assert torch.equal(gradient(False), gradient(True))


def test_checkpointed_loss():
    x, idx, val, _ = _make(6, 3001, 9, "f32")
    head = torch.nn.Linear(16, 3001, device="cuda")
    h = torch.randn(6, 16, device="cuda")

    def loss(h):
        return pd.distill_topk(head(h), idx, val, 1.5)

    want = torch.autograd.grad(loss(h).sum(), head.weight)[0]
    kept = checkpoint(loss, h.clone().requires_grad_(), use_reentrant=False)
    junk = [torch.full((6, 3001), 7.0, device="cuda") for _ in range(4)]  # takes the memory of what was not kept
    assert torch.equal(torch.autograd.grad(kept.sum(), head.weight)[0], want), junk


def test_captured_step():
    """Forward and backward captured together, replayed on new inputs."""
    x, idx, val, lse = _make(8, 32000, 32, "bf16", tail=True)
    y, idy, valy, lsey = _make(8, 32000, 32, "bf16", tail=True, seed=1)
    want = pd.distill_topk_grad(y, idy, valy, teacher_lse=lsey)
    leaf = x.clone().requires_grad_()
    up = torch.ones(8).cuda()
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(pd.distill_topk(leaf, idx, val, teacher_lse=lse), leaf, up)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(g):
        loss = pd.distill_topk(leaf, idx, val, teacher_lse=lse)
        grad, = torch.autograd.grad(loss, leaf, up)
        fused = pd.distill_topk_grad(leaf, idx, val, teacher_lse=lse)
    with torch.no_grad():
        leaf.copy_(y)
        idx.copy_(idy)
        val.copy_(valy)
        lse.copy_(lsey)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(loss, want[0]) and torch.equal(fused[0], want[0]) and torch.equal(fused[1], want[1])
    # the same factor, rounded apart once more
    assert torch.allclose(grad.float(), want[1].float(), rtol=2.0 ** -7, atol=1e-12)


def test_other_stream():
    x, idx, val, _ = _make(16, 128256, 32, "bf16")
    want = pd.distill_topk_grad(x, idx, val)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(5):
        got = pd.distill_topk_grad(x, idx, val, stream=s.cuda_stream)
        s.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_large_strides():
    """Offsets beyond 2^31 elements, in logits and gradient."""
    ld, V, N = (1 << 28) + 1, 1000, 10
    x, idx, val, _ = _make(N, V, 8, "bf16")
    _, want = pd.distill_topk_grad(x, idx, val)
    buf = torch.empty(N * ld, dtype=torch.bfloat16, device="cuda").as_strided((N, V), (ld, 1))
    buf.copy_(x)
    _, got = pd.distill_topk_grad(buf, idx, val, grad=buf)
    # rows of other alignments are added in another order
    assert torch.allclose(got.float(), want.float(), rtol=2.0 ** -7, atol=1e-9)


def test_teacher_lists_from_the_library():
    """The teacher's own lists: top_logprobs at temperature 1 (log sum 0), and a
    student equal to its teacher has loss 0 and no gradient."""
    x = (torch.randn(12, 32001, generator=torch.Generator().manual_seed(9)) * 3).cuda()
    lp, tok, _ = pb.top_logprobs(x, 64)
    zero = torch.zeros(12).cuda()
    loss, grad = pd.distill_topk_grad(x, tok, lp, teacher_lse=zero)
    # f32 log-probabilities of size 20: each off by 2^-24 * 20 + 3e-6, and the tail the rest of it
    assert loss.abs().max() <= 2e-5 and grad.abs().max() <= 2e-5
    _compare(x, tok, lp, 1.0, zero, None, "f32")


def test_empty_batch():
    x = torch.zeros(0, 100, device="cuda")
    idx, val = torch.zeros(0, 4, dtype=torch.int32, device="cuda"), torch.zeros(0, 4, device="cuda")
    loss, grad = pd.distill_topk_grad(x, idx, val)
    assert loss.shape == (0,) and grad.shape == (0, 100)
