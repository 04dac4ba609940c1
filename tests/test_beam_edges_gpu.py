"""Beam search calls that the other tests pass by, against the 64-bit oracle
(oracle/beam.py).  Tolerances are test_beam_gpu.py's unless stated."""
import numpy as np
import pytest
import torch

import beam as OB
import pesti_beam as pb
from test_beam_gpu import DT, NEG, _check, _drive, _logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_log_sums_of_rows_with_nan(dtype):
    """A NaN in a row leaves its log sum as close as the kernel states, 1.95e-6,
    and rounded once to f32.  Every lane adds one term of 1 and terms just below
    half an f32 step of it, each of which a running f32 sum loses."""
    unit = 1024 if dtype == "f32" else 2048
    x = torch.full((3, 2 * unit), -16.75, dtype=DT[dtype], device="cuda")
    x[:, torch.arange(32) * (unit // 256)] = 0.0
    x[1, unit - 1] = float("nan")
    x[2, ::unit - 1] = float("nan")
    lse = torch.empty(3, device="cuda")
    pb.beam_select(x, 1, 4, lse=lse)
    want = np.array([OB.row_logp(r)[1] for r in x.float().cpu().numpy()])
    off = np.abs(lse.cpu().numpy().astype(np.float64) - want)
    assert np.all(off <= 1.95e-6 + np.abs(want) * 2.0 ** -24), off


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("G,lse", [(1, False), (40, False), (60, True)])
def test_equal_candidates_beside_dead_beams(dtype, G, lse):
    """More candidates share the K-th score than are ranked by counting, and some
    beams have no candidates: dead, NaN, masked wholly."""
    W, V, K = 10, 3000, 32 if G == 60 else 64
    x = torch.zeros(G * W, V, dtype=DT[dtype], device="cuda").view(G, W, V)
    x[:, 2] = float("nan")
    x[:, 4] = NEG
    x[:, 5] = 7.0
    cum = torch.zeros(G, W, device="cuda")
    cum[:, 2] = NEG
    cum[:, 7] = float("nan")
    cum[:, 9] = NEG
    got = [pb.beam_select(x.view(G * W, V), W, K, cum=cum, lse=out)
           for out in (None, torch.empty(G * W, device="cuda"))][int(lse)]
    want = OB.select(x[0].float().cpu().numpy(), W, K, cum[:1].cpu().numpy())
    for g in range(G):
        assert np.array_equal(got[1][g].cpu().numpy(), want[1][0])
        assert np.array_equal(got[2][g].cpu().numpy(), want[2][0])
        assert np.all(np.abs(got[0][g].cpu().numpy() - want[0][0]) <= 3e-6 + np.abs(want[0][0]) * 2.0 ** -24)


def test_written_tensors_have_new_versions():
    """A backward pass that needs the old values of what a call overwrote is refused."""
    states = [torch.rand(4, 3, device="cuda"), torch.rand(4, 2, 5, 2, device="cuda")]
    parent = torch.tensor([[1, 0, 3, 2]], dtype=torch.int32, device="cuda")
    for t in states:
        y = torch.ones_like(t, requires_grad=True)
        z = (y * t).sum()
        pb.beam_reorder([t, torch.zeros(4, 1, device="cuda")], parent)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.backward()
    # out of place: the outputs, not the states
    a, b = torch.rand(4, 3, device="cuda"), torch.empty(4, 3, device="cuda")
    before = a._version, b._version, parent._version
    pb.beam_reorder(a, parent, out=b)
    assert a._version == before[0] and b._version > before[1] and parent._version == before[2]

    x, cum = _logits(4, 1000, "f32"), torch.zeros(1, 4, device="cuda")
    out = (torch.empty(1, 8, device="cuda"), *torch.empty(2, 1, 8, dtype=torch.int32, device="cuda"))
    lse = torch.empty(4, device="cuda")
    written, read = (*out, lse), (x, cum)
    before = [t._version for t in (*written, *read)]
    pb.beam_select(x, 4, 8, cum=cum, lse=lse, out=out)
    after = [t._version for t in (*written, *read)]
    assert all(p < q for p, q in zip(before[:4], after[:4])) and before[4:] == after[4:]

    st = pb.BeamState(1, 4, max_tokens=5, max_seq_len=9)
    table = torch.rand(1000, 3, device="cuda", requires_grad=True)
    z = torch.nn.functional.embedding(st.last, table).sum()
    st.advance(*out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    names = ("cum", "last", "parent", "tokens", "count", "done", "fin_tokens", "fin_len", "fin_score", "fin_count")
    before = [getattr(st, n)._version for n in names]
    st.reset()
    assert all(getattr(st, n)._version > v for n, v in zip(names, before))
    with torch.inference_mode():  # tensors without versions
        s = torch.rand(4, 3, device="cuda")
        want = s[[1, 0, 3, 2]]
        assert torch.equal(pb.beam_reorder(s, parent), want)
        st = pb.BeamState(1, 4, max_tokens=5, max_seq_len=9)
        st.advance(*pb.beam_select(x, 4, 8, cum=st.cum, done=st.done, lse=torch.empty(4, device="cuda")))


@pytest.mark.parametrize("kw,code", [
    (dict(max_tokens=0, max_seq_len=0), 3), (dict(max_tokens=7, max_seq_len=0), 3),
    (dict(max_tokens=0, max_seq_len=7), 2),
])
def test_limit_of_nothing(kw, code):
    """A search whose limit is 0 ends at once: 3 where count is max_seq_len, else 2."""
    st, _ = _drive(3, 4, 8, 2, 5, [3], **kw)
    assert st.done.tolist() == [code] * 3 and st.count.tolist() == [0] * 3 and st.fin_count.tolist() == [0] * 3
    assert (st.parent == -1).all()


@pytest.mark.parametrize("G,W,K", [(1, 4, 128), (100, 8, 64), (300, 64, 128)])
def test_many_equal_candidates_many_times(G, W, K):
    """Every candidate of many groups has the same score: lower beams and tokens first, in every call."""
    x = torch.zeros(G * W, 1500, device="cuda")
    token = torch.arange(K, dtype=torch.int32, device="cuda").expand(G, K)
    for _ in range(20):
        _, t, p = pb.beam_select(x, W, K)
        assert torch.equal(t, token) and not p.any()


@pytest.mark.parametrize("G", [1, 30])
def test_equal_candidates_of_few_live_beams(G):
    """Three of 64 beams live, their 384 candidates equal; the rows of the others hold NaN."""
    W, V, K = 64, 1200, 128
    x = torch.full((G, W, V), float("nan"), device="cuda")
    cum = torch.full((G, W), NEG, device="cuda")
    x[:, [5, 31, 63]] = 2.0
    cum[:, [5, 31, 63]] = -1.0
    s, t, p = pb.beam_select(x.view(G * W, V), W, K, cum=cum)
    assert torch.equal(t, torch.arange(K, dtype=torch.int32, device="cuda").expand(G, K)) and (p == 5).all()
    # one rounding to f32 of a sum in 64 bits
    want = -1.0 - float(np.log(V))
    assert (s.double() - want).abs().max() <= abs(want) * 2.0 ** -24 + 1e-12


def test_reorder_beside_its_parents():
    """States that lie next to the parents in one buffer, and states read from them."""
    buf = torch.arange(64, dtype=torch.int32, device="cuda")
    parent = buf[16:24].view(2, 4)
    parent.copy_(torch.tensor([[1, 0, 3, 3], [2, 2, -1, 0]]))
    idx = torch.tensor([1, 0, 3, 3, 6, 6, 6, 4], device="cuda")
    before, behind = buf[:16].view(8, 2), buf[24:].view(8, 5)
    want = before[idx].clone(), behind[idx].clone()
    pb.beam_reorder([before, behind], parent)
    assert torch.equal(before, want[0]) and torch.equal(behind, want[1])
    out = pb.beam_reorder(parent.view(8), parent, out=torch.empty(8, dtype=torch.int32, device="cuda"))
    assert torch.equal(out, parent.view(8)[idx])
    with pytest.raises(Exception, match="parents overlap"):
        pb.beam_reorder(parent.view(8), parent)


def test_the_default_stream_by_its_handle():
    """stream=0 is the legacy default stream, also from within another stream: what a call allocates belongs to it."""
    side, index = torch.cuda.Stream(), torch.cuda.current_device()
    x = _logits(8, 5000, "bf16")
    want = pb.beam_select(x, 4, 8)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        seen = pb._launch(torch.device("cuda", index), 0, lambda st: (st, torch.cuda.current_stream().cuda_stream))
        assert seen == (0, 0)
        assert torch.cuda.current_stream() == side
        got = pb.beam_select(x, 4, 8, stream=0)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
