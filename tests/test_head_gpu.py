"""Cross entropy from hidden states on the GPU against the 64-bit oracle
(oracle/head.py): losses and gradients of both entry points.

Tolerances.  A product over K is summed in f32 in steps of 16: each step is off
by at most one unit in the last place of what has been summed, 2^-23 of the
sum of magnitudes S, and its own 16 products by one more: (K/16 + 4) 2^-22 S
covers both.  d = that for the logits' K = D is also the error of lse, plus
2^-20 for the hardware's 2^x (2^-22.5), the tiles' f32 sums and lse in f32
relative to |lse| <= 30.
  |loss - exact| <= w [2 d (1 + 2 zeta |lse|) + 2^-20 (1 + |lse|)]
A gradient's G = c1 p - c2 - c3 is off by p's error, expm1(2 d + 2^-19), by
the f32 steps 2^-22 of its parts, and by half a step of its type (of up to 64
rows: by that of what half a step leaves); f16 holds it down to 2^-39 of the
largest sum of parts.  Then the product's own sum over K
(padded rows count as rows), and half a step of the result's type."""
import pytest
import torch

import head as OH
import pesti_head as ph

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
TINY = {"bf16": 2.0 ** -120, "f16": 2.0 ** -25}


def _make(N, V, D, dtype, seed=0, pad=0.0, lean=4.0):
    g = torch.Generator(device="cuda").manual_seed(seed * 104729 + N * 31 + V * 7 + D)
    head = torch.randn(V, D, generator=g, device="cuda") * (1.5 / D ** 0.5)
    target = torch.randint(0, V, (N,), generator=g, device="cuda")
    hidden = torch.randn(N, D, generator=g, device="cuda")
    hidden += head[target] * lean * torch.rand(N, 1, generator=g, device="cuda")
    target = torch.where(torch.rand(N, generator=g, device="cuda") < pad, -100, target)
    return hidden.to(DT[dtype]), head.to(DT[dtype]), target


def _step(K):
    return (K / 16 + 4) * 2.0 ** -22


def _close(got, want, tol, what):
    got = got.double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), torch.nonzero(bad)[:4].tolist(), got[bad][:4].tolist(),
                           want[bad][:4].tolist(), tol.expand_as(want)[bad][:4].tolist())


def _compare(hidden, head, target, loss=None, gh=None, gw=None, weight=None, eps=0.0, zeta=0.0, up=None):
    dtype = {v: k for k, v in DT.items()}[hidden.dtype]
    (N, D), V = hidden.shape, head.shape[0]
    o = OH.cross_entropy(hidden, head, target, weight, eps, zeta, up)
    w = torch.ones(N, dtype=torch.float64, device=hidden.device) if weight is None else weight.double().abs()
    d = _step(D) * o["size"]
    if loss is not None:
        assert loss.dtype == torch.float32 and loss.shape == (N,)
        tol = w * (2 * d * (1 + 2 * zeta * o["lse"].abs()) + 2.0 ** -20 * (1 + o["lse"].abs() + zeta * o["lse"] ** 2))
        _close(loss, o["loss"], tol, "loss")
        assert (loss[~o["live"]] == 0).all()
    half = float(torch.finfo(hidden.dtype).eps) / 2
    dG = o["p"] * torch.expm1(2 * d + 2.0 ** -19)[:, None] + 2.0 ** -22 * o["parts"] + (half if N > 64 else half * half) * o["G"].abs()
    if dtype == "f16":
        dG = dG + 2.0 ** -39 * o["parts"].sum(1).max() * o["live"][:, None]
    if gh is not None:
        assert gh.dtype == hidden.dtype and gh.shape == hidden.shape
        tol = (dG + _step(V) * (o["G"].abs() + dG)) @ o["abs_head"]
        _close(gh, o["grad_hidden"], tol + half * (o["grad_hidden"].abs() + tol) + TINY[dtype], "grad_hidden")
        assert (gh[~o["live"]] == 0).all()
    if gw is not None:
        assert gw.dtype == head.dtype and gw.shape == head.shape
        tol = (dG + _step(N) * (o["G"].abs() + dG)).T @ o["abs_hidden"]
        _close(gw, o["grad_head"], tol + half * (o["grad_head"].abs() + tol) + TINY[dtype], "grad_head")


def _all_ways(hidden, head, target, weight=None, eps=0.0, zeta=0.0, up=None):
    """Scoring, loss and gradients in one call, forward and backward."""
    more = dict(weight=weight, label_smoothing=eps, z_loss=zeta)
    score = ph.linear_cross_entropy(hidden, head, target, **more)
    _compare(hidden, head, target, loss=score, weight=weight, eps=eps, zeta=zeta)
    loss, gh, gw = ph.linear_cross_entropy_grad(hidden, head, target, **more)
    assert torch.equal(loss, score)
    _compare(hidden, head, target, gh=gh, gw=gw, weight=weight, eps=eps, zeta=zeta)
    x, y = hidden.detach().requires_grad_(), head.detach().requires_grad_()
    loss = ph.linear_cross_entropy(x, y, target, **more)
    assert torch.equal(loss.detach(), score)
    up = torch.ones(len(target), device="cuda") if up is None else up
    a, b = torch.autograd.grad(loss, (x, y), up)
    _compare(hidden, head, target, gh=a, gw=b, weight=weight, eps=eps, zeta=zeta, up=up)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("N,V,D", [
    (1, 1, 1), (1, 2, 8), (3, 255, 7), (2, 256, 64), (5, 257, 65), (127, 1000, 72), (128, 512, 256), (129, 3001, 257),
    (256, 511, 520), (257, 4099, 136), (300, 32001, 200), (1, 50000, 1000), (700, 1030, 2056),
])
def test_against_the_oracle(dtype, N, V, D):
    hidden, head, target = _make(N, V, D, dtype)
    if D % 8:  # rows of the head begin at multiples of 16 bytes
        head = torch.zeros(V, -(-D // 8) * 8, dtype=head.dtype, device="cuda")[:, :D].copy_(head)
    up = torch.linspace(-1.0, 2.0, N).cuda()
    _all_ways(hidden, head, target, up=up)


@pytest.mark.parametrize("eps,zeta", [(0.1, 0.0), (0.0, 1e-2), (0.3, 1e-3)])
def test_smoothing_and_z_loss(eps, zeta):
    hidden, head, target = _make(150, 2500, 264, "bf16", pad=0.2)
    up = torch.rand(150, device="cuda") - 0.3
    _all_ways(hidden, head, target, eps=eps, zeta=zeta, up=up)
    hidden, head, target = _make(40, 700, 72, "f16")
    _all_ways(hidden, head, target, eps=eps, zeta=zeta, up=up[:40] * 1024)


@pytest.mark.parametrize("kind", [torch.int64, torch.int32])
def test_padding_is_not_read(kind):
    """Rows without a target in [0, V) or with weight 0 hold what must not reach any output."""
    N, V, D = 300, 1500, 136
    hidden, head, target = _make(N, V, D, "bf16", seed=1)
    target[::3] = torch.tensor([-1, -100, V, V + 7], device="cuda").repeat(25)
    if kind == torch.int64:
        target[3] = (1 << 40) + 5
        target[6] = -(1 << 40)
    weight = torch.rand(N, device="cuda") + 0.5
    weight[1::10] = 0.0
    gone = (target < 0) | (target >= V) | (weight == 0)
    weight[0] = float("nan")  # of a row without a target
    clean = hidden.clone()
    clean[gone] = 0
    dirty = hidden.clone()
    dirty[gone] = torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda").to(hidden.dtype).repeat(46)[:D]
    up = torch.rand(N, device="cuda")
    up[0] = float("inf")
    ok = torch.where(gone, 0.0, weight)
    _all_ways(clean, head, target.to(kind), weight=ok, up=torch.where(gone, 0.0, up))
    want = ph.linear_cross_entropy_grad(clean, head, target.to(kind), weight=ok)
    got = ph.linear_cross_entropy_grad(dirty, head, target.to(kind), weight=weight)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x, y = dirty.requires_grad_(), head.requires_grad_()
    a, b = torch.autograd.grad(ph.linear_cross_entropy(x, y, target.to(kind), weight), (x, y), up)
    assert torch.isfinite(a.float()).all() and torch.isfinite(b.float()).all()


@pytest.mark.parametrize("N", [1, 130, 700])
def test_nothing_but_padding(N):
    hidden, head, target = _make(N, 900, 72, "bf16")
    target[:] = -100
    loss, gh, gw = ph.linear_cross_entropy_grad(hidden, head, target)
    for t in (loss, gh, gw):
        assert (t == 0).all()
    x, y = hidden.requires_grad_(), head.requires_grad_()
    a, b = torch.autograd.grad(ph.linear_cross_entropy(x, y, target).sum(), (x, y))
    assert (a == 0).all() and (b == 0).all()


def test_pieces_of_the_vocabulary():
    """Many rows: G is made, used and forgotten piece by piece."""
    hidden, head, target = _make(16500, 20001, 64, "bf16", pad=0.1)
    up = torch.rand(16500, device="cuda")
    _all_ways(hidden, head, target, up=up)


def test_many_rows():
    """More rows than a grid's second dimension."""
    hidden, head, target = _make(70_001, 300, 24, "bf16", pad=0.3)
    _all_ways(hidden, head, target)


def test_long_vocabulary_with_few_rows():
    """K of the hidden states' gradient in many ranges."""
    for N in (2, 200):
        hidden, head, target = _make(N, 300_001, 136, "f16")
        _all_ways(hidden, head, target)


def test_strides_and_alignment():
    """Hidden rows of any stride and alignment, spread head rows: the same bits as packed ones."""
    N, V, D = 140, 1100, 200
    hidden, head, target = _make(N, V, D, "bf16", pad=0.1)
    want = ph.linear_cross_entropy_grad(hidden, head, target)
    h2 = torch.full((N * 211 + 8,), float("nan"), dtype=hidden.dtype, device="cuda")[3:].as_strided((N, D), (211, 1))
    h2.copy_(hidden)
    w2 = torch.full((V, 264), float("nan"), dtype=head.dtype, device="cuda")[:, 8:8 + D]
    w2.copy_(head)
    got = ph.linear_cross_entropy_grad(h2, w2, target)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    up = torch.rand(N, device="cuda")
    a = torch.autograd.grad(ph.linear_cross_entropy(x := hidden.requires_grad_(), y := head.requires_grad_(), target),
                            (x, y), up)
    b = torch.autograd.grad(ph.linear_cross_entropy(x := h2.requires_grad_(), y := w2.requires_grad_(), target),
                            (x, y), up)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # one row for all, and a transposed view of a single row's length
    one = hidden[:1].detach().expand(N, D)
    got = ph.linear_cross_entropy(one, head, target)
    assert torch.equal(got, ph.linear_cross_entropy(one.contiguous(), head, target))


def test_what_not_finite_logits_do():
    hidden, head, target = _make(200, 1000, 64, "bf16")
    hidden[7, 3] = float("nan")
    hidden[150, 0] = float("inf")
    loss, gh, _ = ph.linear_cross_entropy_grad(hidden, head, target)
    bad = torch.zeros(200, dtype=torch.bool, device="cuda")
    bad[[7, 150]] = True
    assert torch.equal(torch.isnan(loss), bad) and torch.equal(torch.isnan(gh.float()).any(1), bad)
    keep = ~bad
    target[bad] = -1
    want = ph.linear_cross_entropy_grad(hidden, head, target)
    assert torch.equal(loss[keep], want[0][keep]) and torch.equal(gh[keep], want[1][keep])
    assert torch.isfinite(want[2].float()).all()


def test_large_logits():
    """Logits of some hundreds: all of the mass on one token, or ties of two."""
    hidden, head, target = _make(64, 777, 128, "bf16", lean=0.0)
    head[5] = head[6]
    hidden[:32] = head[5] * 200
    target[:16] = 5
    _all_ways(hidden, head, target)


def test_one_gradient_alone():
    hidden, head, target = _make(90, 1200, 72, "bf16")
    x, y = hidden.clone().requires_grad_(), head.clone().requires_grad_()
    both = torch.autograd.grad(ph.linear_cross_entropy(x, y, target).sum(), (x, y))
    assert torch.equal(torch.autograd.grad(ph.linear_cross_entropy(x, head, target).sum(), x)[0], both[0])
    assert torch.equal(torch.autograd.grad(ph.linear_cross_entropy(hidden, y, target).sum(), y)[0], both[1])
    assert not ph.linear_cross_entropy(hidden, head, target).requires_grad
    weight = torch.ones(90, device="cuda").requires_grad_()
    assert not ph.linear_cross_entropy(hidden, head, target, weight).requires_grad


def test_upstream_gradients():
    """Expanded, strided and scalar ones; another step of the same graph."""
    hidden, head, target = _make(60, 500, 64, "bf16")
    x = hidden.requires_grad_()
    loss = ph.linear_cross_entropy(x, head, target)
    want, = torch.autograd.grad(loss, x, torch.full((60,), 2.0, device="cuda"), retain_graph=True)
    got, = torch.autograd.grad(loss, x, torch.full((1,), 2.0, device="cuda").expand(60), retain_graph=True)
    assert torch.equal(got, want)
    spread = torch.full((60, 3), 2.0, device="cuda")[:, 1]
    assert torch.equal(torch.autograd.grad(loss, x, spread)[0], want)


def test_against_differences():
    """The loss moves along a direction as the gradient says.  Hidden states and head are perturbed by 1/8 of
    themselves at most, in 64-bit sums of the oracle's own losses at points that bf16 holds exactly."""
    N, V, D = 40, 300, 32
    hidden, head, target = _make(N, V, D, "bf16")
    _, gh, gw = ph.linear_cross_entropy_grad(hidden, head, target, label_smoothing=0.1, z_loss=1e-3)
    for leaf, grad in ((0, gh), (1, gw)):
        base = (hidden, head)[leaf]
        step = (torch.randint(0, 2, base.shape, device="cuda") * 2 - 1).to(torch.float64) * 2.0 ** -12

        def total(sign):
            at = [hidden.double(), head.double()]
            at[leaf] = at[leaf] + sign * step
            return OH.cross_entropy(at[0], at[1], target, eps=0.1, zeta=1e-3)["loss"].sum()

        slope = (total(1) - total(-1)) / 2
        said = (grad.double() * step).sum()
        # bf16 gradients: G and the result half a step each, 2^-8 of sums of magnitudes, and the third derivative
        o = OH.cross_entropy(hidden, head, target, eps=0.1, zeta=1e-3)
        room = (o["G"].abs() @ o["abs_head"], o["G"].abs().T @ o["abs_hidden"])[leaf]
        assert (slope - said).abs() <= 1.1 * 2.0 ** -8 * (room * step.abs()).sum() + 1e-6


def test_the_same_bits_every_time():
    hidden, head, target = _make(333, 9001, 264, "bf16", pad=0.1)
    first = ph.linear_cross_entropy_grad(hidden, head, target)
    for _ in range(5):
        again = ph.linear_cross_entropy_grad(hidden, head, target)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_saved_tensors_may_move():
    hidden, head, target = _make(50, 700, 72, "bf16", pad=0.1)
    weight, up = torch.rand(50, device="cuda"), torch.rand(50, device="cuda")

    def padded(t):
        t = t.detach()
        room = t.new_zeros(t.shape[0], *[n + 8 for n in t.shape[1:]])
        return room[tuple(slice(0, n) for n in t.shape)].copy_(t)

    def gradient(hooks):
        x, y, t, w = (v.clone() for v in (hidden, head, target, weight))
        x.requires_grad_(), y.requires_grad_()
        if not hooks:
            return torch.autograd.grad(ph.linear_cross_entropy(x, y, t, w), (x, y), up)
        with torch.autograd.graph.saved_tensors_hooks(padded, lambda v: v):
            loss = ph.linear_cross_entropy(x, y, t, w)
        with torch.no_grad():
            x.zero_(), y.zero_(), t.zero_(), w.zero_()
        return torch.autograd.grad(loss, (x, y), up)

    assert all(torch.equal(a, b) for a, b in zip(gradient(False), gradient(True)))


def test_overwritten_inputs_have_no_backward():
    hidden, head, target = _make(20, 300, 64, "bf16")
    x = hidden.requires_grad_()
    loss = ph.linear_cross_entropy(x, head, target)
    head.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.sum().backward()


def test_checkpointed_loss():
    _, head, target = _make(30, 900, 64, "bf16")
    up = torch.nn.Linear(16, 64, device="cuda", dtype=torch.bfloat16)
    h = torch.randn(30, 16, device="cuda").bfloat16()

    def loss(h):
        return ph.linear_cross_entropy(up(h), head, target)

    want = torch.autograd.grad(loss(h).sum(), up.weight)[0]
    kept = torch.utils.checkpoint.checkpoint(loss, h.clone().requires_grad_(), use_reentrant=False)
    junk = [torch.full((30, 64), 7.0, device="cuda").bfloat16() for _ in range(4)]
    assert torch.equal(torch.autograd.grad(kept.sum(), up.weight)[0], want), junk


def test_captured_step():
    """Two captured steps that share a pool, replayed on new inputs: also fewer rows than at the capture."""
    hidden, head, target = _make(200, 3000, 136, "bf16")
    h2, w2, t2 = _make(200, 3000, 136, "bf16", seed=1, pad=0.5)
    want = ph.linear_cross_entropy_grad(h2, w2, t2)
    x, y, up = hidden.clone().requires_grad_(), head.clone().requires_grad_(), torch.ones(200, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ph.linear_cross_entropy(x, y, target), (x, y), up)
    torch.cuda.current_stream().wait_stream(side)
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        loss = ph.linear_cross_entropy(x, y, target)
        a, b = torch.autograd.grad(loss, (x, y), up)
    with torch.cuda.graph(two, pool=one.pool()):
        fused = ph.linear_cross_entropy_grad(x.detach(), y.detach(), target)
    with torch.no_grad():
        x.copy_(h2), y.copy_(w2), target.copy_(t2)
    for _ in range(2):
        one.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, want[0]) and torch.equal(a, want[1]) and torch.equal(b, want[2])
        two.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(fused, want))


def test_streams():
    """Another stream by handle, the default one from within another, and two at once."""
    hidden, head, target = _make(300, 20000, 264, "bf16")
    want = ph.linear_cross_entropy_grad(hidden, head, target)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = [ph.linear_cross_entropy_grad(hidden, head, target, stream=s.cuda_stream) for s in streams]
        for s, g in zip(streams, got):
            s.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(g, want))
    with torch.cuda.stream(streams[0]):
        got = ph.linear_cross_entropy_grad(hidden, head, target, stream=0)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_no_rows():
    hidden, head, target = _make(1, 100, 64, "bf16")
    loss, gh, gw = ph.linear_cross_entropy_grad(hidden[:0], head, target[:0])
    assert loss.shape == (0,) and gh.shape == (0, 64) and (gw == 0).all() and gw.shape == (100, 64)
    y = head.requires_grad_()
    g, = torch.autograd.grad(ph.linear_cross_entropy(hidden[:0], y, target[:0]).sum(), y)
    assert (g == 0).all()


def test_offsets_beyond_32_bits():
    """Hidden and head rows that lie 2^31 bytes and more behind the first."""
    N, V, D = 20, 600, 64
    hidden, head, target = _make(N, V, D, "bf16")
    want = ph.linear_cross_entropy_grad(hidden, head, target)
    ld = (1 << 28) + 8
    h2 = torch.empty(N * ld, dtype=torch.bfloat16, device="cuda").as_strided((N, D), (ld, 1))
    h2.copy_(hidden)
    got = ph.linear_cross_entropy_grad(h2, head, target)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del h2
    ld = (1 << 23) + 8
    w2 = torch.empty(V * ld, dtype=torch.bfloat16, device="cuda").as_strided((V, D), (ld, 1))
    w2.copy_(head)
    got = ph.linear_cross_entropy_grad(hidden, w2, target)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_trains():
    """A few steps of a small model through the loss: the gradients of the layer below and of the head are those of
    the same model in plain operations, to the types' steps."""
    g = torch.Generator(device="cuda").manual_seed(3)
    V, D, N = 500, 64, 96
    body = torch.nn.Linear(32, D, device="cuda").bfloat16()
    head = (torch.randn(V, D, generator=g, device="cuda") * 0.1).bfloat16().requires_grad_()
    x = torch.randn(N, 32, generator=g, device="cuda").bfloat16()
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    params = [*body.parameters(), head]
    for _ in range(3):
        h = body(x)
        grads = torch.autograd.grad(ph.linear_cross_entropy(h, head, t).mean(), params)
        o = OH.cross_entropy(h, head, t, up=torch.full((N,), 1.0 / N, device="cuda"))
        want = torch.autograd.grad(body(x), params[:-1], o["grad_hidden"].to(torch.bfloat16))
        for a, b in zip(grads, (*want, o["grad_head"])):
            # G, the gradient of h, and the layer's own product: three roundings of 2^-9 and room for their growth
            assert (a.double() - b.double()).norm() <= 4 * 2.0 ** -8 * b.double().norm()
        with torch.no_grad():
            for p, g_ in zip(params, grads):
                p -= 0.5 * g_


def test_modes():
    """Inference mode, no grad, a head that is a view of a larger table, and no second derivative."""
    hidden, head, target = _make(70, 900, 64, "bf16")
    want = ph.linear_cross_entropy_grad(hidden, head, target)
    with torch.inference_mode():
        assert torch.equal(ph.linear_cross_entropy(hidden, head, target), want[0])
        got = ph.linear_cross_entropy_grad(hidden, head, target)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    table = torch.zeros(1000, 64, dtype=head.dtype, device="cuda")
    table[50:950] = head
    table.requires_grad_()
    loss = ph.linear_cross_entropy(hidden, table[50:950], target)
    g, = torch.autograd.grad(loss.sum(), table)
    assert torch.equal(g[50:950], want[2]) and (g[:50] == 0).all() and (g[950:] == 0).all()
    x = hidden.requires_grad_()
    g, = torch.autograd.grad(ph.linear_cross_entropy(x, head, target).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()
