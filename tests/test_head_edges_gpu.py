"""Cross entropy from hidden states where it can go wrong: confident rows,
rows beside ones that are not finite, saved tensors that come back otherwise,
pairs of blocks on narrow tiles.

Confident rows (p of the target t near 1) against the 64-bit oracle.  Logits
off by d (tests/test_head_gpu.py; here of the at most 1024 of K that are summed
at once, and an addition for each such part) change each G but the target's by
a factor of at most expm1(2 d), beside 2^-22 for the hardware's 2^x and
2^-22 (1 + |lse|) for lse and its product with log2(e) in f32; and so they do
G_t = p_t - 1, minus the sum of the others, if the logits are the very ones that
are in lse.  All further errors of p_t are absolute: ABS."""
import contextlib

import pytest
import torch

import head as OH
import pesti_head as ph
import test_head_gpu as OE

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


def _loss_room(hidden, o):
    """Bound of -log p_t off its definition, relative to itself: the others' sum over the target's exponential, whose
    logits are off by d each, whose 2^x by 2^-22, and which some tens of f32 additions make, 2^-19."""
    D = hidden.shape[1]
    d = (_step(min(D, PART)) + (D // PART) * 2.0 ** -24) * o["size"]
    return torch.expm1(2 * d) + 2.0 ** -19


@pytest.mark.parametrize("way", ["one call", "autograd"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("N,V,D", [(1, 2001, 4096), (40, 2000, 1000), (48, 30_001, 4096), (200, 3000, 4096), (1100, 2000, 520)])
def test_very_confident_rows(way, dtype, N, V, D):
    """1 - p of 1e-2 to 1e-7: losses and gradients are exact relative to themselves, ABS is 0."""
    doubt = torch.logspace(-7, -2, N, device="cuda")
    hidden, head, target = _confident(N, V, D, dtype, doubt)
    o = OH.cross_entropy(hidden, head, target)
    loss = ph.linear_cross_entropy(hidden, head, target)
    _check(loss, o["loss"], (_loss_room(hidden, o) + 2.0 ** -24) * o["loss"], "loss")
    _compare(way, hidden, head, target, 0.0)


def test_a_target_of_any_probability():
    """z_t far above, near and far below the other logits, alone in the vocabulary, and infinite."""
    V, D = 1500, 64
    g = torch.Generator(device="cuda").manual_seed(4)
    head = torch.randn(V, D, generator=g, device="cuda").mul_(0.2).bfloat16()
    for N in (60, 300):
        target = torch.randint(0, V, (N,), generator=g, device="cuda")
        w = head[target].float()
        hidden = (w * torch.linspace(-60, 60, N, device="cuda")[:, None]).bfloat16()
        o = OH.cross_entropy(hidden, head, target)
        got = ph.linear_cross_entropy(hidden, head, target)
        # (the oracle's own loss is a difference of 64-bit numbers)
        _check(got, o["loss"], (_loss_room(hidden, o) + 2.0 ** -24) * o["loss"] + 2.0 ** -50 * (1 + o["lse"].abs()), "loss")
        alone = ph.linear_cross_entropy(hidden, head[:1], torch.zeros_like(target))
        assert (alone == 0).all()
        z = hidden.double() @ head[0].double()
        square = ph.linear_cross_entropy(hidden, head[:1], torch.zeros_like(target), z_loss=0.5, label_smoothing=0.25)
        # z_t is off by d, and its square by 2 z d; loss rounded once
        size = (hidden.double().abs() @ head[0].double().abs())
        assert ((square.double() - 0.5 * z * z).abs() <= z.abs() * _step(D) * size + (_step(D) * size) ** 2 + 2.0 ** -23 * z * z).all()
    hidden = torch.ones(3, D, device="cuda").bfloat16()
    head[7] = float("inf")
    head[8] = -float("inf")
    loss, gh, _ = ph.linear_cross_entropy_grad(hidden, head, torch.tensor([7, 8, 9], device="cuda"))
    assert torch.isnan(loss).all()
    head[7] = 0
    loss = ph.linear_cross_entropy(hidden, head, torch.tensor([7, 8, 9], device="cuda"))
    want = -torch.log_softmax(hidden.double() @ head.double().T, 1)[torch.arange(3), torch.tensor([7, 8, 9])]
    assert loss[1] == float("inf") and torch.allclose(loss[[0, 2]].double(), want[[0, 2]].to(loss.device), rtol=1e-4)
    smooth = ph.linear_cross_entropy(hidden, head, torch.tensor([7, 8, 9], device="cuda"), label_smoothing=0.1)
    assert (smooth == float("inf")).all()


@pytest.mark.parametrize("eps,zeta", [(0.0, 0.0), (0.1, 1e-3)])
def test_gradients_of_an_f32_lse(eps, zeta):
    """pesti_linear_ce and pesti_linear_ce_backward, which pass on no -log p: G_t is off by 2^-22 (1 + |lse|) w up more."""
    import ctypes

    import pesti_sampler as ps
    lib = ps.load_library()
    for N, V, D in ((50, 900, 264), (200, 2000, 520)):
        hidden, head, target = _confident(N, V, D, "bf16", torch.logspace(-1, -4, N, device="cuda"))
        weight, up = torch.rand(N, device="cuda") + 0.5, torch.rand(N, device="cuda") + 0.5
        need = lib.pesti_linear_ce_workspace(ps.PESTI_BF16, N, V, D, 3)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        loss, lse = torch.empty(2, N, device="cuda")
        gh, gw = torch.empty_like(hidden), torch.empty_like(head)
        args = (hidden.data_ptr(), ps.PESTI_BF16, N, D, D, head.data_ptr(), V, D, target.data_ptr(), 8,
                weight.data_ptr(), eps, zeta)
        st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert lib.pesti_linear_ce(*args, loss.data_ptr(), lse.data_ptr(), None, D, None, D, ws.data_ptr(), need, st) == 0
        assert lib.pesti_linear_ce_backward(*args, lse.data_ptr(), up.data_ptr(), 1, gh.data_ptr(), D, gw.data_ptr(), D,
                                            ws.data_ptr(), need, st) == 0
        o = OH.cross_entropy(hidden, head, target, weight, eps, zeta, up)
        assert ((lse.double() - o["lse"]).abs() <= _step(D) * o["size"] + 2.0 ** -20 * (1 + o["lse"].abs())).all()
        o["hot"] = torch.zeros_like(o["G"]).scatter_(1, target[:, None], 1.0)
        # smoothing and z-loss: sums of parts, each off by some units of 2^-24, beside the target's own
        dG = _room(hidden, o, 0.0) + 2.0 ** -22 * o["parts"] + o["hot"] * (2.0 ** -22 * (2 + o["lse"].abs()) * weight.double() * up.double())[:, None]
        dG = dG + torch.expm1(2 * _step(D) * o["size"])[:, None] * o["p"] * (1.0 if eps or zeta else 0.0)
        half = 2.0 ** -8  # a step of bfloat16's 8 bits of mantissa is 2^-7 of the power of two below a value
        tol = (dG + _step(V) * (o["G"].abs() + dG)) @ o["abs_head"]
        _check(gh, o["grad_hidden"], tol + half * (o["grad_hidden"].abs() + tol) + TINY["bf16"], "grad_hidden")
        tol = (dG + _step(N) * (o["G"].abs() + dG)).T @ o["abs_hidden"]
        _check(gw, o["grad_head"], tol + half * (o["grad_head"].abs() + tol) + TINY["bf16"], "grad_head")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("scale", [1e-4, 1.0, 1e5])
@pytest.mark.parametrize("N", [40, 200, 1100])
def test_rows_beside_ones_that_are_not_finite(dtype, scale, N):
    """Rows with NaN or infinite logits, weights or upstream gradients leave the other rows' outputs as they are without
    them: in f16 too, where G is held times a power of two that all rows share."""
    g = torch.Generator(device="cuda").manual_seed(N)
    V, D = 3001, 72
    head = torch.randn(V, D, generator=g, device="cuda").mul_(1.5 / D ** 0.5).to(DT[dtype])
    hidden = torch.randn(N, D, generator=g, device="cuda").to(DT[dtype])
    target = torch.randint(0, V, (N,), generator=g, device="cuda")
    weight = scale * (0.5 + torch.rand(N, generator=g, device="cuda"))
    up = 0.5 + torch.rand(N, generator=g, device="cuda")
    bad = torch.zeros(N, dtype=torch.bool, device="cuda")
    bad[[7, 20, 33]] = True
    clean = torch.where(bad, -1, target)
    ill = weight.clone()
    ill[33] = float("inf")
    dirty = hidden.clone()
    dirty[7, 3], dirty[20, 0] = float("nan"), float("inf")
    want = ph.linear_cross_entropy_grad(hidden, head, clean, weight)
    loss, gh, _ = ph.linear_cross_entropy_grad(dirty, head, target, ill)
    assert torch.isnan(loss[[7, 20]]).all() and not torch.isfinite(loss[33])
    assert torch.equal(loss[~bad], want[0][~bad]) and torch.equal(gh[~bad], want[1][~bad])
    o = OH.cross_entropy(hidden, head, clean, weight)
    if dtype == "bf16" or scale < 1e4:
        assert torch.isfinite(gh[~bad].float()).all()
        assert ((gh.double() - o["grad_hidden"]).norm(dim=1) <= 2.0 ** -7 * o["grad_hidden"].norm(dim=1))[~bad].all()

    def backward(h, t, w, u):
        x, y = h.detach().requires_grad_(), head.detach().requires_grad_()
        return torch.autograd.grad(ph.linear_cross_entropy(x, y, t, w), (x, y), u)

    u2 = up.clone()
    u2[20] = float("nan")
    u2[33] = float("inf")
    want = backward(hidden, clean, weight, up)
    got = backward(dirty, target, weight, u2)
    assert torch.equal(got[0][~bad], want[0][~bad])


@pytest.mark.parametrize("pin", [False, True])
@pytest.mark.parametrize("V,D", [(300, 1001), (1, 1001), (300, 1000), (37, 1)])
def test_saved_on_the_host(V, D, pin):
    """Saved tensors come back without the room behind their rows."""
    g = torch.Generator(device="cuda").manual_seed(D)
    N = 50
    room = torch.full((V, -(-D // 8) * 8), float("nan"), device="cuda").bfloat16()
    head = room[:, :D].copy_(torch.randn(V, D, generator=g, device="cuda") / D ** 0.5)
    hidden = torch.randn(N, D, generator=g, device="cuda").bfloat16()
    target = torch.randint(0, V, (N,), generator=g, device="cuda")
    weight, up = torch.rand(2, N, generator=g, device="cuda")

    def gradient(saved):
        x, y = hidden.detach().requires_grad_(), head.detach().requires_grad_()
        with saved:
            loss = ph.linear_cross_entropy(x, y, target, weight)
        return torch.autograd.grad(loss, (x, y), up)

    want = gradient(contextlib.nullcontext())
    got = gradient(torch.autograd.graph.save_on_cpu(pin_memory=pin))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_saved_elsewhere():
    """A head that comes back at another alignment, or by columns."""
    g = torch.Generator(device="cuda").manual_seed(2)
    N, V, D = 30, 200, 64
    head = (torch.randn(V, D, generator=g, device="cuda") / 8).bfloat16()
    hidden = torch.randn(N, D, generator=g, device="cuda").bfloat16()
    target = torch.randint(0, V, (N,), generator=g, device="cuda")

    def moved(t):
        t = t.detach()
        return t.new_empty(t.numel() + 4)[4:].copy_(t.reshape(-1)).view(t.shape)

    def turned(t):
        t = t.detach()
        return t.t().contiguous().t() if t.dim() == 2 else t.clone()

    def gradient(pack):
        x, y = hidden.detach().requires_grad_(), head.detach().requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            loss = ph.linear_cross_entropy(x, y, target)
        return torch.autograd.grad(loss.sum(), (x, y))

    want = gradient(lambda t: t)
    for pack in (moved, turned):
        assert all(torch.equal(a, b) for a, b in zip(gradient(pack), want))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("N,V", [(200, 20000), (1024, 3001), (700, 20000), (500, 50000), (200, 50257), (1000, 5000)])
def test_pairs_on_narrow_tiles(dtype, N, V):
    """More than 128 rows on tiles of 144, 176, 208 and 240 columns, an odd multiple of 16: each block of a pair copies
    half a tile, whose rows are no multiple of 16."""
    hidden, head, target = OE._make(N, V, 64, dtype, pad=0.1)
    OE._all_ways(hidden, head, target, eps=0.1, zeta=1e-3, up=torch.rand(N, device="cuda") + 0.5)


@pytest.mark.parametrize("N", [20, 200])
@pytest.mark.parametrize("scale", [1e33, 1e36, 3e38])
def test_weights_near_the_end_of_f32(N, scale):
    """f16 gradients of rows of any finite weight: where the other factor is 0, 0, and beyond f16 infinite, but not NaN."""
    g = torch.Generator(device="cuda").manual_seed(N)
    V, D = 500, 64
    head = torch.randn(V, D, generator=g, device="cuda").div_(8).half()
    hidden = torch.randn(N, D, generator=g, device="cuda").half()
    target = torch.randint(0, V, (N,), generator=g, device="cuda")
    head[:, 5] = 0
    hidden[:, 7] = 0
    weight = torch.full((N,), scale, device="cuda")
    # (G's own bound, twice the weight, has to be finite)
    _, gh, gw = ph.linear_cross_entropy_grad(hidden, head, target, weight / 2)
    assert (gh[:, 5] == 0).all() and (gw[:, 7] == 0).all()
    assert not torch.isnan(gh).any() and not torch.isnan(gw).any()
