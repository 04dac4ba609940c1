"""What the vocabulary projection's entry points refuse, before any device work
(no GPU needed), and their oracle."""
import pytest
import torch

import head as OH
import pesti_head as ph
import pesti_sampler as ps

BAD = ps.PESTI_E_INVALID_ARG
P = 1 << 20   # addresses that are never used: every call below is refused first
Q = 1 << 40
R = 1 << 42
S = 1 << 44


@pytest.fixture(scope="module")
def lib():
    return ps.load_library()


CE = dict(hidden=P, dtype=ps.PESTI_BF16, N=4, D=64, h_ld=64, head=Q, V=100, w_ld=64, target=P, target_bytes=8,
          weight=None, eps=0.0, zeta=0.0)
FORWARD = dict(loss=P, lse=None, gh=None, gh_ld=64, gw=None, gw_ld=64, ws=P, ws_bytes=1 << 40, stream=None)
BACKWARD = dict(lse=P, up=P, up_stride=1, gh=R, gh_ld=64, gw=S, gw_ld=64, ws=P, ws_bytes=1 << 40, stream=None)

COMMON = [
    (dict(dtype=ps.PESTI_F32), "bf16 or f16"), (dict(dtype=ps.PESTI_FP8_E4M3), "bf16 or f16"), (dict(N=-1), "N < 0"),
    (dict(N=(1 << 24) + 1), "N must"), (dict(V=0), "V must"), (dict(V=(1 << 24) + 1), "V must"), (dict(D=0), "D must"),
    (dict(D=(1 << 20) + 1, h_ld=1 << 21, w_ld=1 << 21), "D must"), (dict(h_ld=-64), "negative stride"),
    (dict(w_ld=56), "w_ld is below"), (dict(w_ld=100), "multiple of 8"), (dict(target_bytes=2), "4 or 8 bytes"),
    (dict(eps=-0.1), "label_smoothing"), (dict(eps=1.0), "label_smoothing"), (dict(eps=float("nan")), "label_smoothing"),
    (dict(zeta=-1.0), "z_loss"), (dict(zeta=float("nan")), "z_loss"), (dict(zeta=float("inf")), "z_loss"),
    (dict(hidden=None), "null hidden"), (dict(head=None), "null hidden"), (dict(target=None), "null hidden"),
    (dict(hidden=P + 1), "hidden states are not aligned"), (dict(head=Q + 8), "16-byte"),
    (dict(target=P + 4), "targets are not"), (dict(weight=P + 2), "weights are not"),
    (dict(gh=R, gh_ld=63), "dh_ld is below"), (dict(gh=R + 1), "not aligned"), (dict(gw=S, gw_ld=56), "dw_ld is below"),
    (dict(gw=S, gw_ld=65), "multiple of 8"), (dict(gw=S + 8), "16-byte"), (dict(gh=P), "overlap"),
    (dict(gw=Q), "overlap"), (dict(gh=R, gw=R), "gradients overlap"), (dict(gh=Q + 12800 - 64), "overlap"),
    (dict(ws=None), "workspace too small"), (dict(ws_bytes=100), "workspace too small"), (dict(ws=P + 16), "256-byte"),
]


@pytest.mark.parametrize("change,msg", COMMON + [
    (dict(loss=None), "null loss"), (dict(loss=P + 2), "loss or lse is not"), (dict(lse=P + 1), "loss or lse is not"),
])
def test_forward_refusals(lib, change, msg):
    assert lib.pesti_linear_ce(*{**CE, **FORWARD, **change}.values()) == BAD
    assert msg in lib.pesti_last_error().decode()


@pytest.mark.parametrize("change,msg", COMMON + [
    (dict(lse=None), "null lse"), (dict(up=None), "null lse"), (dict(up_stride=-1), "negative stride"),
    (dict(gh=None, gw=None), "no gradient"), (dict(lse=P + 2), "gradient is not aligned"),
    (dict(up=P + 1), "gradient is not aligned"),
])
def test_backward_refusals(lib, change, msg):
    assert lib.pesti_linear_ce_backward(*{**CE, **BACKWARD, **change}.values()) == BAD
    assert msg in lib.pesti_last_error().decode()


def test_workspace(lib):
    f = lib.pesti_linear_ce_workspace
    small = f(ps.PESTI_BF16, 1, 1000, 64, 1)
    assert 0 < small < f(ps.PESTI_BF16, 1, 1000, 64, 3) and f(ps.PESTI_BF16, 0, 1000, 64, 3) >= 0
    for bad in ((ps.PESTI_F32, 1, 10, 8, 1), (ps.PESTI_BF16, -1, 10, 8, 1), (ps.PESTI_BF16, 1, 0, 8, 1),
                (ps.PESTI_BF16, 1, 10, 0, 1), (ps.PESTI_BF16, 1, 10, 8, 0), (ps.PESTI_BF16, 1, 10, 8, 4)):
        assert f(*bad) == BAD
    # far below the logits: 2^16 rows of 256000 are 31 GB in bf16
    assert f(ps.PESTI_BF16, 1 << 16, 256000, 4096, 3) < 8 << 30
    assert lib.pesti_linear_ce(*{**CE, **FORWARD, "N": 0}.values()) == ps.PESTI_OK
    assert lib.pesti_linear_ce_backward(*{**CE, **BACKWARD, "N": 0, "gw": None}.values()) == ps.PESTI_OK


HELD = dict(q=Q, scale=R, V=100, D=300, group=64)


@pytest.mark.parametrize("change,msg", [
    (dict(dtype=ps.PESTI_FP8_E5M2), "f32, bf16 or f16"), (dict(V=0), "V must"), (dict(V=(1 << 24) + 1), "V must"),
    (dict(D=0), "D must"), (dict(D=(1 << 20) + 1, ld=1 << 21), "D must"), (dict(group=16), "group must"),
    (dict(group=0), "group must"), (dict(q=None), "null weights"), (dict(scale=None), "null weights"),
    (dict(q=Q + 8), "16-byte"), (dict(scale=R + 2), "16-byte"), (dict(ld=299), "ld is below"), (dict(head=None), "null"),
    (dict(head=P + 2), "not aligned"), (dict(head=Q), "overlap"), (dict(head=R), "overlap"), (dict(scale=Q), "overlap"),
])
def test_conversion_refusals(lib, change, msg):
    a = {**dict(head=P, dtype=ps.PESTI_F32, ld=300), **HELD, **change}
    there = [a[k] for k in ("head", "dtype", "V", "D", "ld", "group", "q", "scale")] + [None]
    back = [a[k] for k in ("q", "scale", "V", "D", "group", "head", "dtype", "ld")] + [None]
    for rc in (lib.pesti_q4_quantize(*there), lib.pesti_q4_dequantize(*back)):
        assert rc == BAD
        assert msg in lib.pesti_last_error().decode()


LOGITS = dict(x=P, dtype=ps.PESTI_BF16, B=30, D=300, x_ld=300, q=Q, scale=R, V=100, group=64, logits=S,
              out=ps.PESTI_F32, ld=100, ws=P, ws_bytes=1 << 30, stream=None)


@pytest.mark.parametrize("change,msg", [
    (dict(dtype=ps.PESTI_FP8_E4M3), "f32, bf16 or f16"), (dict(out=ps.PESTI_FP8_E4M3), "logits must be"),
    (dict(B=-1), "B < 0"), (dict(B=(1 << 24) + 1), "B must"), (dict(D=0), "D must"), (dict(V=0), "V must"),
    (dict(group=48), "group must"), (dict(x_ld=-300), "negative stride"), (dict(ld=99), "ld is below"),
    (dict(q=None), "null weights"), (dict(scale=None), "null weights"), (dict(x=None), "null x"),
    (dict(logits=None), "null x"), (dict(q=Q + 4), "16-byte"), (dict(scale=R + 8), "16-byte"),
    (dict(x=P + 1), "x is not aligned"), (dict(logits=S + 2), "logits are not aligned"), (dict(logits=P), "overlap"),
    (dict(logits=Q + 16), "overlap"), (dict(logits=R + 16), "overlap"), (dict(ws=None), "workspace too small"),
    (dict(ws_bytes=100), "workspace too small"), (dict(ws=P + 64), "256-byte"),
])
def test_logits_refusals(lib, change, msg):
    assert lib.pesti_q4_logits(*{**LOGITS, **change}.values()) == BAD
    assert msg in lib.pesti_last_error().decode()
    assert lib.pesti_q4_logits(*{**LOGITS, "B": 0}.values()) == ps.PESTI_OK


def test_python_refusals():
    h, w, t = torch.zeros(4, 64).bfloat16(), torch.zeros(10, 64).bfloat16(), torch.zeros(4, dtype=torch.int64)
    for args, msg in [
        ((h.float(), w.float(), t), "bfloat16 or both float16"), ((h, w.half(), t), "bfloat16 or both float16"),
        ((h[0], w, t), r"\[N, D\]"), ((h, w[:, :32], t), r"\[N, D\]"), ((h, w, t[:3]), "target"),
        ((h, w, t.short()), "target"), ((h, w, t[:1].expand(4)), "target"), ((h.t().contiguous().t(), w, t), "rows of"),
        ((h, w.t().contiguous().t(), t), "rows of"), ((h, w, t, torch.ones(4).double()), "weight"),
        ((h, w, t, torch.ones(3)), "weight"), ((h, w, t), "CUDA device"),
    ]:
        with pytest.raises(ValueError, match=msg):
            ph.linear_cross_entropy(*args)
        with pytest.raises(ValueError, match=msg):
            ph.linear_cross_entropy_grad(*args)
    for args, msg in [((w[0],), "head must"), ((w.int(),), "head must"), ((w.t(), 32), "contiguous"),
                      ((w, 48), "group"), ((w,), "CUDA device")]:
        with pytest.raises(ValueError, match=msg):
            ph.quantize_head(*args)
    held = ph.QuantizedHead(torch.zeros(1, 1, 64, 64, dtype=torch.uint8), torch.zeros(1, 1, 64, 2).bfloat16(), 10, 64, 64)
    assert held.V == 10 and held.scale.shape == (10, 1)
    for change, msg in [(dict(V=0), "at least 1"), (dict(group=16), "group"), (dict(V=65), "packed must"),
                        (dict(D=129), "packed must"), (dict(packed=held.packed.int()), "packed must"),
                        (dict(group=32), "tile_scale must"), (dict(tile_scale=held.tile_scale.float()), "tile_scale must"),
                        (dict(packed=torch.zeros(1, 1, 64, 64, dtype=torch.uint8).transpose(2, 3)), "packed must")]:
        with pytest.raises(ValueError, match=msg):
            ph.QuantizedHead(**{**dict(packed=held.packed, tile_scale=held.tile_scale, V=10, D=64, group=64), **change})
    for args, msg in [((h[0], held), "x must"), ((h.int(), held), "x must"), ((h[:, :32], held), "different D"),
                      ((h.t().contiguous().t(), held), "contiguous"), ((h, held, torch.int32), "dtype must"),
                      ((h, held, None, torch.zeros(4, 9)), "out must"), ((h, held), "CUDA device")]:
        with pytest.raises(ValueError, match=msg):
            ph.head_logits(*args)
    for kw, msg in [(dict(dtype=torch.int8), "dtype must"), (dict(out=torch.zeros(9, 64)), "out must"),
                    (dict(), "CUDA device")]:
        with pytest.raises(ValueError, match=msg):
            held.dequantize(**kw)


def test_the_oracle():
    """The oracle's gradients are autograd's, and its 4-bit weights are no further off than half a step."""
    g = torch.Generator().manual_seed(0)
    h = torch.randn(6, 10, generator=g, dtype=torch.float64).requires_grad_()
    w = torch.randn(20, 10, generator=g, dtype=torch.float64).requires_grad_()
    t = torch.tensor([0, 19, -100, 20, 3, 3])
    weight, up = torch.rand(6, generator=g) + 0.1, torch.rand(6, generator=g)
    weight[4] = 0
    o = OH.cross_entropy(h, w, t, weight, 0.1, 1e-2, up)
    live = torch.tensor([0, 1, 5])
    z = h[live] @ w.T
    loss = torch.nn.functional.cross_entropy(z, t[live], reduction="none", label_smoothing=0.1)
    loss = weight[live].double() * (loss + 1e-2 * torch.logsumexp(z, 1) ** 2)
    gh, gw = torch.autograd.grad((loss * up[live].double()).sum(), (h, w))
    assert torch.allclose(o["loss"][live], loss) and o["loss"][[2, 3, 4]].abs().max() == 0
    assert torch.allclose(o["grad_hidden"], gh) and torch.allclose(o["grad_head"], gw)
    w = torch.randn(7, 100, generator=g)
    q, scale = OH.quantize(w, 32)
    assert scale.shape == (7, 4) and q.min() >= -8 and q.max() <= 7
    s = scale.double().abs().repeat_interleave(32, 1)[:, :100]
    # values beyond 7 steps of the scale are cut to 7; the scale itself is off by 2^-9
    assert ((OH.held_values(q, scale, 32) - w.double()).abs() <= torch.where(q == 7, 1.04 * s, 0.5 * s)).all()
