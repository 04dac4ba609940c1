"""Cross entropy from hidden states where it can go wrong: confident rows.

Confident rows (p of the target t near 1) against the 64-bit oracle.  Logits
off by d (tests/test_head_gpu.py, here of the parts of at most 1024 of K that
are summed at once, and an addition for each part) change each G but the target's by a factor
of at most expm1(2 d), beside 2^-22 for the hardware's 2^x and 2^-22 (1 + |lse|)
for lse and its product with log2(e) in f32, and so does G_t = p_t - 1, minus the sum of the others, if the logits are
the very ones that are in lse.  All further errors of p_t are absolute: ABS."""
import pytest
import torch

import head as OH
import pesti_head as ph

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
TINY = {"bf16": 2.0 ** -120, "f16": 2.0 ** -25}
PART = 1024  # of K


def _confident(N, V, D, dtype, doubt):
    """Rows whose target's logit exceeds the rest by what leaves them 1 - p of about doubt[n]; their targets differ."""
    g = torch.Generator(device="cuda").manual_seed(N * 31 + V * 7 + D)
    head = (torch.randn(V, D, generator=g, device="cuda") * (1.5 / D ** 0.5)).to(DT[dtype])
    target = torch.randperm(V, generator=g, device="cuda")[:N]
    w = head[target].double()
    z = torch.log(V / doubt)[:, None]
    return (w * (z / (w * w).sum(1, keepdim=True))).to(DT[dtype]), head, target


def _step(K):
    return (K / 16 + 4) * 2.0 ** -22


def _check(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol)
    worst = ((got.double() - want).abs() / tol).max().item()
    assert not bad.any(), (what, int(bad.sum()), torch.nonzero(bad)[:4].tolist(), "worst %.3g of the bound" % worst)


def _room(hidden, o, absolute):
    """Bound of |G| off its definition, the target's by `absolute` besides."""
    N, D = hidden.shape
    half = float(torch.finfo(hidden.dtype).eps) / 2
    d = (_step(min(D, PART)) + (D // PART) * 2.0 ** -24) * o["size"]
    off = torch.expm1(2 * d) + 2.0 ** -22 * (2 + o["lse"].abs()) + (half if N > 64 else half * half)
    room = off[:, None] * o["G"].abs()
    if hidden.dtype == torch.float16:
        room = room + 2.0 ** -39 * o["parts"].sum(1).max()
    return room + absolute * o["hot"]


def _gradients(way, hidden, head, target):
    if way == "one call":
        return ph.linear_cross_entropy_grad(hidden, head, target)[1:]
    x, y = hidden.detach().requires_grad_(), head.detach().requires_grad_()
    return torch.autograd.grad(ph.linear_cross_entropy(x, y, target).sum(), (x, y))


def _compare(way, hidden, head, target, absolute):
    dtype = {v: k for k, v in DT.items()}[hidden.dtype]
    (N, D), V = hidden.shape, head.shape[0]
    o = OH.cross_entropy(hidden, head, target)
    o["hot"] = torch.zeros_like(o["G"]).scatter_(1, target[:, None], 1.0)
    gh, gw = _gradients(way, hidden, head, target)
    half = float(torch.finfo(hidden.dtype).eps) / 2
    dG = _room(hidden, o, absolute)
    tol = (dG + _step(V) * (o["G"].abs() + dG)) @ o["abs_head"]
    _check(gh, o["grad_hidden"], tol + half * (o["grad_hidden"].abs() + tol) + TINY[dtype], "grad_hidden")
    tol = (dG + _step(N) * (o["G"].abs() + dG)).T @ o["abs_hidden"]
    _check(gw, o["grad_head"], tol + half * (o["grad_head"].abs() + tol) + TINY[dtype], "grad_head")


@pytest.mark.parametrize("way", ["one call", "autograd"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("N,V,D", [(1, 2001, 4096), (48, 2000, 4096), (200, 3000, 4096), (33, 1000, 8192)])
def test_confident_rows(way, dtype, N, V, D):
    """ABS: lse and its product with log2(e) are rounded to f32 (2^-24 of themselves each), sums of a tile's exponentials
    and 2^x to f32 (some units of 2^-24 each): 2^-22 (2 + |lse|), at |lse| < 22."""
    doubt = torch.logspace(-2, -4, N, device="cuda")
    _compare(way, *_confident(N, V, D, dtype, doubt), 2.0 ** -22 * 24)
