"""The vocabulary projection's tensor core kernels when a wait on the device gives up: what is not finished is NaN, never
plausible or left unwritten, and the next call is right.  (pesti_testing_give_up; each of these kernels ends by its
waits' own limits, after a second or two.)"""
import contextlib

import pytest
import torch

import pesti_head as ph
import pesti_sampler as ps

pytestmark = pytest.mark.gpu

LOGITS, G, HEAD, HIDDEN, Q4 = range(5)


@contextlib.contextmanager
def _giving_up(product, round):
    lib = ps.load_library()
    assert lib.pesti_testing_give_up(product, round) == 0
    try:
        yield
        torch.cuda.synchronize()
    finally:
        assert lib.pesti_testing_give_up(product, -1) == 0


def _inputs(N, V, D):
    g = torch.Generator(device="cuda").manual_seed(N)
    head = (torch.randn(V, D, generator=g, device="cuda") / D ** 0.5).bfloat16()
    hidden = torch.randn(N, D, generator=g, device="cuda").bfloat16()
    return hidden, head, torch.randint(0, V, (N,), generator=g, device="cuda")


def _sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("N", [40, 200])
def test_the_heads_gradient_alone(N):
    """The last product, with nothing behind it that could tell: its tiles from the third round on are NaN."""
    blocks = 1 if N <= 128 else 2
    D, tile = 264, 128 * blocks
    rounds, units = 4, _sms() // blocks
    V = (rounds * units // 2 - 3) * tile - 5
    hidden, head, target = _inputs(N, V, D)
    y = head.requires_grad_()

    def gradient():
        return torch.autograd.grad(ph.linear_cross_entropy(hidden, y, target).sum(), y)[0]

    want = gradient()
    assert torch.isfinite(want.float()).all()
    with _giving_up(HEAD, 2):
        got = gradient()
    # two tiles of columns to a tile of rows, next to one another
    bad = torch.zeros(V, D, dtype=torch.bool, device="cuda")
    bad[units * tile:] = True
    lost = torch.isnan(got.float())
    # (a block that begins after another's wait has given up makes NaN of all its tiles)
    assert lost[bad].all() and torch.equal(got[~lost], want[~lost])
    assert torch.equal(gradient(), want)


@pytest.mark.parametrize("N,product", [(40, LOGITS), (40, G), (40, HIDDEN), (200, LOGITS), (200, G), (200, HIDDEN)])
def test_products_before_others(N, product):
    """Whatever comes of an unfinished product is NaN, wholly."""
    hidden, head, target = _inputs(N, 3000, 520)
    want = ph.linear_cross_entropy_grad(hidden, head, target)
    with _giving_up(product, 0):
        loss, gh, gw = ph.linear_cross_entropy_grad(hidden, head, target)
    assert torch.isnan(gh.float()).all()
    assert product == HIDDEN or torch.isnan(gw.float()).all()
    assert product != LOGITS or torch.isnan(loss).all()
    got = ph.linear_cross_entropy_grad(hidden, head, target)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("B,dtype", [(20, torch.bfloat16), (64, torch.float32)])
def test_logits(B, dtype):
    """Rows of the weight from the second round of a slot on."""
    per_round = 2 * _sms() * 128
    V, D = 2 * per_round + 1000, 640
    g = torch.Generator(device="cuda").manual_seed(B)
    held = ph.quantize_head(torch.randn(V, D, generator=g, device="cuda").bfloat16(), 64)
    x = torch.randn(B, D, generator=g, device="cuda").to(dtype)
    want = ph.head_logits(x, held)
    with _giving_up(Q4, 1):
        got = ph.head_logits(x, held)
    assert torch.isnan(got[:, per_round:]).all() and torch.equal(got[:, :per_round], want[:, :per_round])
    assert torch.equal(ph.head_logits(x, held), want)
