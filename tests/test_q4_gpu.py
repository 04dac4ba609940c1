"""The 4-bit projection on the GPU against the 64-bit oracle (oracle/head.py):
what is held and read back, bit for bit; logits; a whole decode step.

Tolerance of logits.  Products of x and q are exact.  A group's sum and the sum
over groups in f32: each of the D/16 steps of the products off by at most one
unit of what has been summed and one of its own, 2^-22 of the sum of
magnitudes S; each of the D/g scaled additions by 2^-23 S, and joins of up to 8
parts by 2^-22 S: (D/16 + D/g + 8) 2^-22 S, and half a step of the result's
type (2^-25 for f16's subnormals)."""
import pytest
import torch

import head as OH
import pesti_beam as pb
import pesti_head as ph
import pesti_sampler as ps

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _weight(V, D, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + V * 31 + D)
    w = torch.randn(V, D, generator=g, device="cuda") * 0.02
    w *= torch.where(torch.rand(D, generator=g, device="cuda") < 0.03, 8.0, 1.0)
    return w.to(DT[dtype])


def _check_held(head, group):
    held = ph.quantize_head(head, group)
    V, D = head.shape
    q, scale = OH.quantize(head, group)
    assert torch.equal(held.scale, scale) and held.scale.shape == (V, -(-D // group))
    assert torch.equal(OH.unpack(held.packed, V, D).double(), q)
    want = OH.held_values(q, scale, group)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        assert torch.equal(held.dequantize(dtype), want.float().to(dtype))
    return held, want


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("V,D", [(1, 1), (3, 31), (2, 128), (17, 129), (33, 1000), (130, 2048), (5, 4097)])
def test_held_and_read_back(dtype, group, V, D):
    _check_held(_weight(V, D, dtype), group)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_ties_and_edges(dtype):
    """Equal magnitudes of both signs, quotients at halves and next to them, zeros, tiny and huge groups."""
    t = DT[dtype]
    w = torch.zeros(8, 128, device="cuda")
    w[0, ::2], w[0, 1::2] = 1.0, -1.0
    w[1, ::2], w[1, 1::2] = -1.0, 1.0
    halves = torch.arange(-17, 17, device="cuda").float() / 16.0  # multiples of a half of the scale 1/8
    w[2, :34] = halves
    w[2, 64:98] = -halves * 2
    w[3, 40] = 2.0 ** -13
    w[4] = torch.randn(128, device="cuda") * (2.0 ** -14 if dtype == "f16" else 1e-38)
    w[5] = torch.randn(128, device="cuda").clamp(-3, 3) * (2e4 if dtype == "f16" else 1e38)
    w[6, :8] = torch.tensor([0.0, -0.0, 1e-7, -1e-7, 3.0, -3.0, 2.9999, -2.9999], device="cuda")
    w[7] = 5.0
    w = w.to(t)
    if dtype == "f32":  # one step of f32 to either side of a half
        near = torch.nextafter(w[2], torch.full_like(w[2], 9.0))
        w = torch.cat([w, near[None], torch.nextafter(w[2], torch.full_like(w[2], -9.0))[None]])
    for group in (32, 64, 128):
        _check_held(w, group)


def test_tiny_scales():
    """Scales among bfloat16's subnormals and below."""
    w = torch.randn(16, 64, device="cuda") * torch.logspace(-45, -33, 16, device="cuda")[:, None]
    held = ph.quantize_head(w, 32)
    q, scale = OH.quantize(w, 32)
    # m / -8 of a subnormal f32 is rounded once more, to f32's steps of 2^-149, far below bfloat16's of 2^-133
    assert torch.equal(held.scale, scale)
    assert torch.equal(OH.unpack(held.packed, 16, 64).double(), q)


def test_groups_that_are_not_finite():
    w = _weight(4, 256, "f32")
    w[1, 70], w[2, 3], w[3, 255] = float("nan"), float("inf"), -float("inf")
    got = ph.quantize_head(w, 64).dequantize(torch.float32)
    want = OH.held_values(*OH.quantize(torch.nan_to_num(w, nan=1.0, posinf=1.0, neginf=1.0), 64), 64).float()
    bad = torch.zeros(4, 256, dtype=torch.bool, device="cuda")
    bad[1, 64:128], bad[2, :64], bad[3, 192:] = True, True, True
    assert torch.equal(torch.isnan(got), bad) and torch.equal(got[~bad], want[~bad])
    for rows in (2, 20):
        logits = ph.head_logits(torch.ones(rows, 256, device="cuda"), ph.quantize_head(w, 64))
        assert torch.isnan(logits[:, 1:]).all() and torch.isfinite(logits[:, 0]).all()


@pytest.mark.parametrize("B", [3, 20])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_scales_of_all_magnitudes(B, dtype):
    """Groups of a row that are 2^-60 to 2^60 of one another.  With more rows, scales below 2^-25 of the largest of their
    columns lose bits: an element q s is off by at most 2^-25 steps of what f16 holds, 2^-36 of the largest s, and no
    more than half of itself."""
    V, D, group = 200, 1500, 32
    w = _weight(V, D, "f32")
    n = -(-D // group)
    sizes = torch.exp2(torch.randint(-30, 31, (V, n), generator=torch.Generator().manual_seed(B)).float()).cuda()
    w = w * sizes.repeat_interleave(group, 1)[:, :D]
    held, want = _check_held(w, group)
    x = torch.randn(B, D, generator=torch.Generator().manual_seed(9)).to(DT[dtype]).cuda()
    got = ph.head_logits(x, held, dtype=torch.float32).double()
    exact, S = x.double() @ want.T, x.double().abs() @ want.abs().T
    tol = (D / 16 + D / group + 8) * 2.0 ** -22 * S
    tol = tol + 2.0 ** -36 * x.double().abs().sum(1, keepdim=True) * held.scale.double().abs().amax(1)[None]
    assert ((got - exact).abs() <= tol + 2.0 ** -24 * exact.abs()).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_strided_weights(dtype):
    head = _weight(50, 300, dtype)
    want = ph.quantize_head(head, 32)
    room = torch.full((50, 311), float("nan"), dtype=head.dtype, device="cuda")[:, 5:305]
    room.copy_(head)
    got = ph.quantize_head(room, 32)
    assert torch.equal(got.packed, want.packed) and torch.equal(got.tile_scale, want.tile_scale)
    out = torch.full((50, 311), 7.0, dtype=head.dtype, device="cuda")
    version = out._version
    got.dequantize(out=out[:, 5:305])
    assert out._version > version
    assert torch.equal(out[:, 5:305], want.dequantize(head.dtype))
    assert (out[:, :5] == 7).all() and (out[:, 305:] == 7).all()


def _check_logits(x, held, want, dtype, **more):
    got = ph.head_logits(x, held, dtype=dtype, **more)
    exact = x.double() @ want.T
    S = x.double().abs() @ want.abs().T
    D = x.shape[1]
    half = float(torch.finfo(dtype).eps) / 2
    tol = (D / 16 + D / held.group + 8) * 2.0 ** -22 * S
    tol = tol + half * (exact.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126)
    bad = ~((got.double() - exact).abs() <= tol)
    assert got.dtype == dtype and not bad.any(), (int(bad.sum()), torch.nonzero(bad)[:4].tolist())
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("B,V,D", [
    (1, 1, 1), (1, 33, 130), (2, 1000, 512), (7, 31, 2048), (8, 4099, 700), (9, 257, 1000), (17, 640, 384),
    (33, 2001, 129), (64, 512, 4096), (65, 100, 256), (150, 333, 1300),
])
def test_logits(dtype, group, B, V, D):
    held, want = _check_held(_weight(V, D, "bf16"), group)
    x = torch.randn(B, D, generator=torch.Generator().manual_seed(B)).to(DT[dtype]).cuda()
    a = _check_logits(x, held, want, torch.float32)
    b = _check_logits(x, held, want, torch.bfloat16)
    assert torch.equal(b, a.to(torch.bfloat16))
    assert torch.equal(ph.head_logits(x, held, dtype=torch.float16), a.to(torch.float16))


@pytest.mark.parametrize("B", [3, 20])
@pytest.mark.parametrize("V", [18_900, 19_000, 37_900, 40_000, 76_001])
def test_rounds(B, V):
    """More rows of the weight than all SMs hold at once, and last rounds that fill some of them."""
    held, want = _check_held(_weight(V, 256, "bf16"), 64)
    x = torch.randn(B, 256, generator=torch.Generator().manual_seed(V)).bfloat16().cuda()
    _check_logits(x, held, want, torch.float32)


@pytest.mark.parametrize("B,dtype", [(1, "bf16"), (6, "f32"), (8, "f16"), (20, "bf16"), (33, "f32")])
@pytest.mark.parametrize("V", [63, 64, 65, 127, 128, 129, 191, 193])
@pytest.mark.parametrize("D", [2047, 2048])
def test_tile_edges(B, dtype, V, D):
    """Rows that end inside, at and just behind a tile and a pair of them."""
    held, want = _check_held(_weight(V, D, "bf16"), 64)
    assert held.packed.shape == ((V + 63) // 64, 16, 64, 64)
    x = torch.randn(B, D, generator=torch.Generator().manual_seed(V)).to(DT[dtype]).cuda()
    room = torch.full((B, V + 130), 7.0, device="cuda")
    _check_logits(x, held, want, torch.float32, out=room[:, 1:1 + V])
    assert (room[:, 0] == 7).all() and (room[:, 1 + V:] == 7).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,D", [
    (8, 6272), (8, 6273), (8, 12544), (8, 12545), (4, 12544), (4, 12673), (1, 100_352), (1, 100_353), (3, 70_000),
])
def test_long_rows(dtype, B, D):
    """x at, and just above, what is held in shared memory."""
    held, want = _check_held(_weight(40, D, "bf16"), 128)
    x = torch.randn(B, D, generator=torch.Generator().manual_seed(D)).to(DT[dtype]).cuda()
    _check_logits(x, held, want, torch.float32)


@pytest.mark.parametrize("B", [1, 5, 64])
def test_wide_values_of_x(B):
    """f32 rows of all magnitudes, f16 subnormals, bf16 extremes, infinities and NaN."""
    held, want = _check_held(_weight(70, 600, "f32"), 32)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(B, 600, generator=g) * torch.logspace(-30, 30, 600)
    _check_logits(x.cuda(), held, want, torch.float32)
    _check_logits((torch.randn(B, 600, generator=g) * 2.0 ** -20).half().cuda(), held, want, torch.float32)
    _check_logits((torch.randn(B, 600, generator=g) * 1e36).bfloat16().cuda(), held, want, torch.float32)
    for dtype in DT.values():
        y = torch.randn(B, 600, generator=g).to(dtype).cuda()
        plain = ph.head_logits(y, held, dtype=torch.float32)
        y[B - 1, 9] = float("inf")
        got = ph.head_logits(y, held, dtype=torch.float32)
        assert torch.equal(got[:B - 1], plain[:B - 1])
        q = OH.quantize(_weight(70, 600, "f32"), 32)[0][:, 9]
        s = ph.quantize_head(_weight(70, 600, "f32"), 32).scale[:, 0].double()
        assert torch.equal(torch.isnan(got[B - 1]), q == 0)  # 0 times infinity
        assert torch.equal(got[B - 1][q != 0].double(), (q * s)[q != 0].sign() * float("inf"))
        y[B - 1, 9] = float("nan")
        got = ph.head_logits(y, held, dtype=torch.float32)
        assert torch.isnan(got[B - 1]).all() and torch.equal(got[:B - 1], plain[:B - 1])


def test_strided_x_and_logits():
    held, want = _check_held(_weight(333, 1000, "bf16"), 64)
    x = torch.randn(6, 1000, device="cuda")
    plain = _check_logits(x, held, want, torch.float32)
    room = torch.full((6, 1017), float("nan"), device="cuda")[:, 3:1003]
    room.copy_(x)
    out = torch.full((6, 401), 7.0, device="cuda")
    version = out._version
    got = ph.head_logits(room, held, out=out[:, 1:334])
    assert got.data_ptr() == out[:, 1:334].data_ptr() and out._version > version
    assert torch.equal(got, plain) and (out[:, 0] == 7).all() and (out[:, 334:] == 7).all()
    assert torch.equal(ph.head_logits(x[:1].expand(6, 1000), held), plain[:1].expand(6, 333))


def test_rows_do_not_depend_on_their_batch():
    held = ph.quantize_head(_weight(2000, 1024, "bf16"), 64)
    x = torch.randn(64, 1024, device="cuda").bfloat16()
    whole = ph.head_logits(x, held, dtype=torch.float32)
    for rows in (1, 3, 12, 20, 40):
        got = ph.head_logits(x[:rows], held, dtype=torch.float32)
        # the same products, joined in another order at most: two sums' errors
        S = x[:rows].double().abs() @ held.dequantize(torch.float32).double().abs().T
        assert ((got - whole[:rows]).abs().double() <= 2 * (1024 / 16 + 1024 / 64 + 8) * 2.0 ** -22 * S).all()


def test_no_rows():
    held = ph.quantize_head(_weight(40, 64, "bf16"), 64)
    assert ph.head_logits(torch.zeros(0, 64, device="cuda"), held).shape == (0, 40)


def test_captured_and_on_other_streams():
    held = ph.quantize_head(_weight(3000, 512, "bf16"), 64)
    x, y = torch.randn(2, 4, 512, device="cuda").bfloat16()
    want = ph.head_logits(y, held)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [ph.head_logits(y, held, stream=s.cuda_stream) for s in streams]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    g = torch.cuda.CUDAGraph()
    x = x.contiguous()
    with torch.cuda.graph(g):
        logits = ph.head_logits(x, held)
        again = ph.quantize_head(held.dequantize(torch.float32), 64)
    x.copy_(y)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(logits, want)
    assert torch.equal(again.dequantize(torch.float32), held.dequantize(torch.float32))


def test_offsets_beyond_32_bits():
    """A weight whose elements, and logits whose elements, pass 2^31."""
    V, D = 700_000, 4096
    w = torch.empty(V, D, dtype=torch.bfloat16, device="cuda")
    part = _weight(1000, D, "bf16")
    for a in range(0, V, 1000):
        w[a:a + 1000] = part
    held = ph.quantize_head(w, 128)
    del w
    want = ph.quantize_head(part, 128)
    assert torch.equal(held.scale.view(700, 1000, -1), want.scale.expand(700, 1000, -1))
    x = torch.randn(1, D, device="cuda").bfloat16()
    # K may be shared out otherwise for another V: two sums of the same products, each off by the bound above
    back = want.dequantize(torch.float32).double()
    room = 2 * (D / 16 + D / 128 + 8) * 2.0 ** -22 * (x.double().abs() @ back.abs().T)
    got, one = (ph.head_logits(x, h, dtype=torch.float32).double() for h in (held, want))
    assert ((got.view(700, 1000) - one).abs() <= room).all()
    out = torch.empty(4 * ((1 << 30) + 1), dtype=torch.bfloat16, device="cuda").as_strided((4, 1000), ((1 << 30) + 1, 1))
    x = torch.randn(4, D, device="cuda").bfloat16()
    assert torch.equal(ph.head_logits(x, want, out=out), ph.head_logits(x, want))
    back = held.dequantize(torch.bfloat16)
    assert torch.equal(back[-1000:], want.dequantize(torch.bfloat16))


def test_a_whole_step(sampler):
    """Train the head a little, hold it in 4 bits, and answer from hidden states: sampling, beams, scoring."""
    g = torch.Generator(device="cuda").manual_seed(11)
    V, D, B = 4099, 256, 12
    head = (torch.randn(V, D, generator=g, device="cuda") * 0.1).bfloat16()
    hidden = torch.randn(B, D, generator=g, device="cuda").bfloat16()
    target = torch.randint(0, V, (B,), generator=g, device="cuda")
    for _ in range(3):
        _, _, gw = ph.linear_cross_entropy_grad(hidden, head, target, weight=torch.full((B,), 1.0 / B, device="cuda"))
        head -= 4.0 * gw
    held = ph.quantize_head(head, 32)
    logits = ph.head_logits(hidden, held, dtype=torch.float32)
    cfg, u = ps.SamplingConfig(temperature=0.8, top_p=1.0, top_k=20), torch.rand(B, generator=g, device="cuda")
    assert torch.equal(sampler.sample_hidden(hidden, held, cfg, u), sampler.sample_batch(logits, cfg, u))
    many = sampler.sample_hidden(hidden, held, [cfg] * B, u, kept_width=8)
    assert all(torch.equal(a, b) for a, b in zip(many, sampler.sample_batch(logits, [cfg] * B, u, kept_width=8)))
    score, token, parent = pb.beam_select(logits, 4, 8)
    assert (parent >= 0).all()
    # a beam's score is what scoring its token with the held weight gives: f32 sums of either kind
    back = held.dequantize(torch.bfloat16)
    rows = (torch.arange(3, device="cuda")[:, None] * 4 + parent).reshape(-1)
    exact = ph.head_logits(hidden, ph.quantize_head(back, 32), dtype=torch.float32)
    said = ph.linear_cross_entropy(hidden[rows], back, token.reshape(-1))
    o = OH.cross_entropy(hidden[rows], back, token.reshape(-1))
    want = OH.cross_entropy(hidden[rows], held.dequantize(torch.float32), token.reshape(-1))
    # a score is a logit less the logarithm of a sum of them, each off by the bound at the top of this file; the sum is
    # off by 2e-6 of itself, and scores of up to 70 are rounded to f32 twice
    S = (hidden.double().abs() @ held.dequantize(torch.float32).double().abs().T).amax()
    room = float(2 * (D / 16 + D / 32 + 8) * 2.0 ** -22 * S + 2e-6 + 70 * 2.0 ** -23)
    assert want["loss"].max() < 70 and torch.allclose(-score.reshape(-1).double(), want["loss"], rtol=0, atol=room)
    assert torch.allclose(said.double(), o["loss"], rtol=0, atol=float(2 * (D / 16 + 4) * 2.0 ** -22 * o["size"].max()) + 2e-5)
    assert exact.shape == logits.shape


def test_modes(sampler):
    """Inference mode, tensors that require gradients, and outputs whose old values a backward pass needs."""
    head = _weight(300, 256, "bf16")
    x = torch.randn(5, 256, device="cuda").bfloat16()
    held = ph.quantize_head(head.clone().requires_grad_(), 64)
    want = ph.head_logits(x, held)
    with torch.inference_mode():
        assert torch.equal(ph.head_logits(x, ph.quantize_head(head, 64)), want)
        out = torch.empty(5, 300, device="cuda", dtype=torch.bfloat16)
        assert torch.equal(ph.head_logits(x, held, out=out), want)
        back = torch.empty(300, 256, device="cuda")
        assert torch.equal(held.dequantize(out=back), held.dequantize(torch.float32))
        u = torch.rand(5, device="cuda")
        a = sampler.sample_hidden(x, held, ps.SamplingConfig(top_k=5, top_p=1.0), u)
    assert torch.equal(a, sampler.sample_hidden(x, held, ps.SamplingConfig(top_k=5, top_p=1.0), u))
    got = ph.head_logits(x.requires_grad_(), held)
    assert not got.requires_grad and torch.equal(got, want)
    out = torch.randn(5, 300, device="cuda", requires_grad=True)
    loss = (out * out).sum()
    ph.head_logits(x, held, out=out.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
