"""Beam search on the GPU against the 64-bit oracle (oracle/beam.py): selection,
loop control, reordering of states, and a whole search.

Tolerance of a score: the row's log sum is off by at most 3e-6 (above the bound
that the kernel's own comment derives), and the score is rounded once to f32 (half a
step, 2^-24 of it).  Tokens and parents are exact."""
import numpy as np
import pytest
import torch

import beam as OB
import pesti_beam as pb

pytestmark = pytest.mark.gpu

NEG = -np.inf
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _logits(rows, V, dtype, pad=0, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed * 7919 + rows * 31 + V)
    buf = (torch.randn(rows, V + pad, generator=g) * scale).to(DT[dtype]).cuda()
    return buf[:, :V]


def _check(x, W, K, cum=None, done=None):
    """beam_select of x against the oracle."""
    want = OB.select(x.float().cpu().numpy(), W, K, None if cum is None else cum.cpu().numpy(),
                     None if done is None else done.cpu().numpy())
    lse = torch.full((x.shape[0],), 7.0, device="cuda")
    for with_lse in (False, True):
        s, t, p = pb.beam_select(x, W, K, cum=cum, done=done, lse=lse if with_lse else None)
        s, t, p = s.cpu().numpy().astype(np.float64), t.cpu().numpy(), p.cpu().numpy()
        assert np.array_equal(t, want[1])
        assert np.array_equal(p, want[2])
        with np.errstate(invalid="ignore"):
            off = np.abs(s - want[0])
        fine = np.isfinite(want[0]) & (np.abs(want[0]) < 3e38)
        assert np.array_equal(s == NEG, want[0].astype(np.float32) == NEG)
        assert np.all(off[fine] <= 3e-6 + np.abs(want[0][fine]) * 2.0 ** -24)
    got = lse.cpu().numpy().astype(np.float64)
    fine = np.isfinite(want[3])
    assert np.array_equal(got[~fine], want[3][~fine])
    assert np.all(np.abs(got[fine] - want[3][fine]) <= 3e-6 + np.abs(want[3][fine]) * 2.0 ** -24)
    return s, t, p


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("G,W,V,K,pad", [
    (1, 1, 1, 1, 0), (2, 3, 7, 6, 1), (1, 4, 1000, 8, 0), (3, 5, 4099, 10, 1), (2, 16, 32001, 32, 3),
    (1, 64, 2100, 128, 0), (1, 2, 128256, 4, 0), (4, 2, 2048, 128, 0), (1, 7, 100, 128, 5), (5, 1, 32000, 64, 0),
    (1, 3, 2049, 1, 7), (2, 2, 3, 20, 0), (1, 33, 5000, 100, 1), (3, 9, 40000, 27, 0), (70, 8, 3000, 16, 0),
    (400, 3, 2500, 6, 0), (300, 1, 9000, 40, 0),
])
def test_select(dtype, G, W, V, K, pad):
    x = _logits(G * W, V, dtype, pad)
    g = torch.Generator().manual_seed(V)
    cum = (-5.0 * torch.rand(G, W, generator=g)).cuda()
    _check(x, W, K, cum)
    _check(x, W, K)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_select_very_long_rows(dtype):
    """Rows whose segment maxima are taken in runs."""
    V = 1_300_003 if dtype == "bf16" else 650_001
    x = _logits(2, V, dtype, 1)
    _check(x, 2, 16, torch.tensor([[0.0, -0.5]]).cuda())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_select_masks(dtype):
    """Rows that a mask leaves nothing of, one token of, and few tokens of; NaN
    and +inf; masks of the type's lowest value; dead, NaN and unequal beams."""
    W, V, K = 10, 5003, 20
    x = _logits(W, V, dtype).contiguous()
    x[0] = NEG
    x[1] = NEG
    x[1, 4711] = -2.0
    x[2] = NEG
    x[2, 17::1001] = torch.arange(len(range(17, V, 1001))).to(x.dtype).cuda()
    x[3, ::3] = float("nan")
    x[4, 99] = float("inf")
    x[4, 4000] = float("inf")
    x[5] = torch.finfo(x.dtype).min
    x[6, 1:] = torch.finfo(x.dtype).min
    x[7] = float("nan")
    cum = torch.tensor([[-1.0, -1.5, -2.0, -0.5, -30.0, -4.0, -2.5, -1.0, NEG, float("nan")]]).cuda()
    _check(x, W, K, cum)
    _check(x, W, 128, cum)
    # every row by itself
    _check(x, 1, 8)
    _check(x, 1, 128)


def test_select_dead_groups_and_beams():
    G, W, V, K = 6, 4, 3000, 8
    x = _logits(G * W, V, "f32")
    cum = torch.zeros(G, W).cuda()
    cum[1] = NEG            # every beam dead
    cum[2, 1:] = NEG        # a first step
    done = torch.tensor([0, 0, 0, 1, 0, 255], dtype=torch.uint8).cuda()
    x[3 * W:4 * W] = float("nan")
    s, t, p = _check(x, W, K, cum, done)
    for g in (1, 3, 5):
        assert (s[g] == NEG).all() and (t[g] == -1).all() and (p[g] == -1).all()
    assert (p[2] == 0).all()
    s2, t2, _ = pb.beam_select(x, W, K, cum=cum, done=done != 0)
    assert np.array_equal(t2.cpu().numpy(), t)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("K", [1, 16, 128])
def test_select_ties(dtype, K):
    """Constant rows, few values, sorted rows, equal beams: lower tokens and
    lower beams first, however many share a value."""
    V = 9001
    x = torch.zeros(8, V, dtype=DT[dtype]).cuda()
    x[1] = torch.arange(V).cuda().div(3, rounding_mode="floor").neg().to(x.dtype)        # falling, in steps
    x[2] = torch.arange(V).cuda().to(x.dtype)                                            # rising
    x[3] = (torch.arange(V).cuda() % 3).to(x.dtype)
    x[4] = -0.0
    x[4, ::2] = 0.0
    x[5] = x[6] = _logits(1, V, dtype)[0]
    x[7, 5000:] = 1.0
    _check(x, 1, K)
    cum = torch.tensor([[0.0, 0.0, 0.0, 0.0, 0.0, -1.0, -1.0, 0.0]]).cuda()
    _check(x, 8, K, cum)
    _check(x, 8, K)


@pytest.mark.parametrize("shift", [0.0, 1e-7, 4e-7, 2e-6])
def test_select_orders_near_ties(shift):
    """Beams whose candidates are closer than the sums' own error: equal rows
    with scores a few f32 steps apart, at different alignments."""
    V, W, K = 30011, 6, 24
    buf = torch.zeros(W, V + 2).cuda()
    buf[:, :V] = _logits(1, V, "f32", seed=5)
    cum = (torch.tensor([[3.0, 1.0, 5.0, 0.0, 4.0, 2.0]]) * shift).cuda()
    _check(buf[:, :V], W, K, cum)


def test_select_large_strides():
    """Offsets beyond 2^31 elements and 2^32 bytes."""
    ld, V, W = (1 << 28) + 1, 1000, 10
    buf = torch.empty(W * ld, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((W, V), (ld, 1))
    x.copy_(_logits(W, V, "bf16"))
    _check(x, W, 16, torch.zeros(1, W).cuda())


def test_top_logprobs():
    x = _logits(9, 32001, "bf16", 1)
    lp, tok, lse = pb.top_logprobs(x, 50)
    want = torch.log_softmax(x.double(), 1)
    top = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :50]
    assert torch.equal(tok.long(), top)
    assert (lp.double() - want.gather(1, top)).abs().max() <= 3e-6 + 40 * 2.0 ** -24
    assert (lse.double() - torch.logsumexp(x.double(), 1)).abs().max() <= 3e-6 + 40 * 2.0 ** -24


def _drive(G, W, K, steps, seed, stop, **kw):
    """Random candidates through BeamState and the oracle, compared after every step."""
    rng = np.random.default_rng(seed)
    st = pb.BeamState(G, W, stop_tokens=stop, **kw)
    ref = [OB.Beams(W, kw["max_tokens"], kw["max_seq_len"], stop, kw.get("length_penalty", 1.0),
                    kw.get("early_stop", False)) for _ in range(G)]
    for step in range(steps):
        score = -np.sort(rng.random((G, K)) * 3, axis=1).astype(np.float32) - np.float32(0.3 * step)
        token = rng.integers(0, 12, (G, K)).astype(np.int32)
        parent = rng.integers(0, W, (G, K)).astype(np.int32)
        score[rng.random((G, K)) < 0.1] = score[0, 0]  # equal scores in the pool
        cut = rng.integers(0, 3 * K, G)
        for g in range(G):
            score[g, cut[g]:], token[g, cut[g]:], parent[g, cut[g]:] = NEG, -1, -1
        parent[rng.random((G, K)) < 0.02] = W  # outside the group: passed over
        st.advance(*(torch.from_numpy(a).cuda() for a in (score, token, parent)))
        for g in range(G):
            ref[g].advance(score[g], token[g], parent[g])
        have = {n: getattr(st, n).cpu().numpy() for n in ("cum", "last", "parent", "tokens", "count", "done",
                                                          "fin_tokens", "fin_len", "fin_score", "fin_count")}
        for g, r in enumerate(ref):
            assert have["done"][g] == r.done and have["count"][g] == r.count, (step, g)
            assert list(have["parent"][g]) == r.parent
            assert np.array_equal(have["cum"][g], np.array(r.cum, np.float32))
            assert list(have["last"][g]) == r.last
            assert have["fin_count"][g] == len(r.pool)
            for i, (s, toks) in enumerate(r.pool):
                assert have["fin_len"][g, i] == len(toks)
                assert list(have["fin_tokens"][g, i, :len(toks)]) == toks
                # one rounding to f32 on each side of pow and division in 64 bits
                assert abs(float(have["fin_score"][g, i]) - float(s)) <= abs(float(s)) * 2.0 ** -23
            for w in range(W):
                assert list(have["tokens"][g, w, :r.limit]) == r.hist[w]
    return st, ref


@pytest.mark.parametrize("G,W,K,kw", [
    (1, 1, 1, dict(max_tokens=5, max_seq_len=9)),
    (7, 4, 8, dict(max_tokens=20, max_seq_len=20, length_penalty=0.8)),
    (5, 4, 8, dict(max_tokens=300, max_seq_len=280, length_penalty=0.0, early_stop=True)),
    (3, 64, 128, dict(max_tokens=9, max_seq_len=400, length_penalty=-0.5)),
    (6, 3, 9, dict(max_tokens=0, max_seq_len=4)),
    (9, 8, 16, dict(max_tokens=400, max_seq_len=150, length_penalty=2.0)),
])
def test_advance(G, W, K, kw):
    steps = min(kw["max_tokens"], kw["max_seq_len"], 160) + 2
    st, ref = _drive(G, W, K, steps, G * 100 + W, [3, 7], **kw)
    assert st.active() == sum(r.done == 0 for r in ref)
    for have, r in zip(st.hypotheses(), ref):
        assert sorted(t for _, t in have) == sorted(t for _, t in r.pool)
        assert [s for s, _ in have] == sorted((s for s, _ in have), reverse=True)


def test_advance_without_stop_tokens_and_reset():
    st, ref = _drive(2, 3, 6, 7, 1, [], max_tokens=5, max_seq_len=64)
    assert set(st.done.tolist()) <= {1, 2}
    st.reset()
    assert st.active() == 2 and st.count.tolist() == [0, 0]
    assert torch.isneginf(st.cum[:, 1:]).all() and (st.cum[:, 0] == 0).all() and (st.parent == -1).all()


@pytest.mark.parametrize("G,W", [(3, 1), (5, 8), (2, 40)])
def test_select_scores_in_place(G, W):
    x = _logits(G * W, 5003, "bf16", seed=4)
    cum = -torch.rand(G, W, device="cuda") * 3
    want = pb.beam_select(x, W, W, cum=cum.clone())
    token, parent = torch.empty(2, G, W, dtype=torch.int32, device="cuda")
    got = pb.beam_select(x, W, W, cum=cum, out=(cum, token, parent))
    assert got[0] is cum and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("device", [0, "cuda", "cuda:0", torch.device("cuda")])
def test_state_devices(device):
    st = pb.BeamState(2, 3, 4, 8, device=device)
    assert st.device == torch.device("cuda", 0) and st.active() == 2


def _permuted(x, parent, W):
    n = x.shape[0]
    idx = [g * W + (p if 0 <= p < W else w) for g, line in enumerate(parent.tolist()) for w, p in enumerate(line)]
    assert len(idx) == n
    return x[torch.tensor(idx, device=x.device)]


@pytest.mark.parametrize("W", [1, 2, 4, 5, 8, 16, 17, 64])
@pytest.mark.parametrize("in_place", [False, True])
def test_reorder(W, in_place):
    G = 3
    g = torch.Generator().manual_seed(W)
    parent = torch.randint(-1, W + 1, (G, W), generator=g).to(torch.int32).cuda()
    mk = lambda *s, dt=torch.float32: torch.randint(0, 200, s, generator=g).to(dt).cuda()  # noqa: E731
    n = G * W
    states = [mk(n, 3, 40, 8, dt=torch.bfloat16)[:, :, :17], mk(n, 5), mk(n), mk(n, 7, dt=torch.uint8),
              mk(n, 33, dt=torch.float16), mk(n, 2, dt=torch.int64), mk(n, 2, 9, 3, dt=torch.uint8)[:, :, 1:4],
              mk(n, 1300), mk(n, 4, 2, 260)[:, 1:, 1:].squeeze(2), mk(n, 0)]
    want = [_permuted(s, parent, W).clone() for s in states]
    if in_place:
        got = pb.beam_reorder(states, parent)
        assert all(a is b for a, b in zip(got, states))
    else:
        keep = [s.clone() for s in states]
        out = [torch.zeros(s.shape, dtype=s.dtype, device=s.device) for s in states]
        out[0] = torch.zeros(n, 3, 40, 8, dtype=torch.bfloat16, device="cuda")[:, :, :17]
        out[6] = torch.zeros(n, 2, 9, 3, dtype=torch.uint8, device="cuda")[:, :, 2:5]
        out[8] = torch.zeros(n, 3, 300, device="cuda")[:, :, :260]
        got = pb.beam_reorder(states, parent, out=out)
        for a, b in zip(states, keep):
            assert torch.equal(a, b)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_reorder_leaves_the_rest():
    """Positions behind the used ones and rows of finished groups stay as they were."""
    x = torch.arange(4 * 2 * 10 * 4, dtype=torch.float32).reshape(4, 2, 10, 4).cuda()
    keep = x.clone()
    parent = torch.tensor([[1, 0], [-1, -1]], dtype=torch.int32).cuda()
    pb.beam_reorder(x[:, :, :6], parent)
    assert torch.equal(x[:, :, 6:], keep[:, :, 6:]) and torch.equal(x[2:], keep[2:])
    assert torch.equal(x[0, :, :6], keep[1, :, :6]) and torch.equal(x[1, :, :6], keep[0, :, :6])


def test_reorder_many_states_and_one():
    states = [torch.full((2, 3), float(i)).cuda() for i in range(150)]
    for i, s in enumerate(states):
        s[1] += 1000 + i
    want = [s.flip(0) for s in states]
    parent = torch.tensor([[1, 0]], dtype=torch.int32).cuda()
    pb.beam_reorder(states, parent)
    assert all(torch.equal(a, b) for a, b in zip(states, want))
    one = pb.beam_reorder(states[0], parent)
    assert one is states[0] and torch.equal(one, want[0].flip(0))
    with pytest.raises(Exception, match="twice"):
        pb.beam_reorder([one, one], parent)


def test_reorder_large_strides():
    """Rows more than 2^31 bytes apart."""
    row = (1 << 30) + 512
    x = torch.empty(5 * row, dtype=torch.uint8, device="cuda")
    v = x.as_strided((5, 3, 1000), (row, 700_000_000 // 2, 1))
    v.copy_(torch.randint(0, 255, (5, 3, 1000), dtype=torch.uint8))
    parent = torch.tensor([[4, 0, 3, 1, 1]], dtype=torch.int32).cuda()
    want = _permuted(v, parent, 5).clone()
    pb.beam_reorder(v, parent)
    assert torch.equal(v, want)


def _search(V, G, W, steps, graph):
    """A whole search over a fixed table of transitions, on the device."""
    g = torch.Generator().manual_seed(11)
    table = (torch.randn(V, V, generator=g) * 2).cuda()
    stop = [1]
    st = pb.BeamState(G, W, max_tokens=steps, max_seq_len=100, stop_tokens=stop, length_penalty=0.7)
    st.last.copy_(torch.arange(G * W).view(G, W) % V)
    start = st.last.clone()
    cache = torch.zeros(G * W, 2, steps, 4, device="cuda")  # what each beam has seen, per position
    pos = torch.zeros(1, dtype=torch.int64, device="cuda")

    def step():
        cache.scatter_(2, pos.view(1, 1, 1, 1).expand(G * W, 2, 1, 4),
                       st.last.view(-1, 1, 1, 1).expand(G * W, 2, 1, 4).float())
        logits = table[st.last.view(-1).long()]
        score, token, parent = pb.beam_select(logits, W, 2 * W, cum=st.cum, done=st.done)
        st.advance(score, token, parent)
        pb.beam_reorder(cache, st.parent)
        pos.add_(1)

    if graph:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            step()
        st.reset()
        st.last.copy_(start)
        cache.zero_()
        pos.zero_()
        for _ in range(steps):
            cg.replay()
    else:
        for _ in range(steps):
            step()
    torch.cuda.synchronize()
    return table.cpu().numpy(), start.cpu().numpy(), st, cache


@pytest.mark.parametrize("graph", [False, True])
def test_search(graph):
    V, G, W, steps = 37, 5, 4, 12
    table, start, st, cache = _search(V, G, W, steps, graph)
    ref = [OB.Beams(W, steps, 100, [1], 0.7) for _ in range(G)]
    seen = [[[] for _ in range(W)] for _ in range(G)]
    for g, r in enumerate(ref):
        r.last = list(map(int, start[g]))
    for _ in range(steps):
        for g, r in enumerate(ref):
            seen[g] = [h + [r.last[w]] for w, h in enumerate(seen[g])]
            # the device holds scores in f32
            cum = np.array([r.cum], np.float32)
            s, t, p, _ = OB.select(table[r.last], W, 2 * W, cum, [r.done])
            r.advance(s[0].astype(np.float32), t[0], p[0])
            seen[g] = [seen[g][p] if p >= 0 else seen[g][w] for w, p in enumerate(r.parent)]
    done = st.done.tolist()
    hyp = st.hypotheses()
    for g, r in enumerate(ref):
        assert done[g] == r.done
        want = sorted(r.pool, key=lambda h: -h[0])
        assert [t for _, t in hyp[g]] == [t for _, t in want]
        # scores: each step adds at most the selection's tolerance
        assert np.allclose([s for s, _ in hyp[g]], [s for s, _ in want], atol=steps * 1e-5, rtol=0)
        assert np.array_equal(cache[g * W:(g + 1) * W, 1, :, 2].cpu().numpy(), np.array(seen[g], np.float32))


def test_other_streams_and_overlapping_calls():
    """Calls on two streams at once, each with its own scratch, by `stream` and
    by the current stream."""
    a, b = _logits(8, 128256, "bf16", seed=1), _logits(8, 128256, "bf16", seed=2)
    cum = torch.zeros(2, 4).cuda()
    want = [[t.clone() for t in pb.beam_select(x, 4, 8, cum=cum)] for x in (a, b)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        one = pb.beam_select(a, 4, 8, cum=cum, stream=s1.cuda_stream)
        with torch.cuda.stream(s2):
            two = pb.beam_select(b, 4, 8, cum=cum)
        s1.synchronize()
        s2.synchronize()
        for got, ref in ((one, want[0]), (two, want[1])):
            assert all(torch.equal(x, y) for x, y in zip(got, ref))


def test_two_captured_graphs_at_once():
    x = [_logits(16, 32000, "f32", seed=s) for s in (3, 4)]
    cum = torch.zeros(4, 4).cuda()
    want = [[t.clone() for t in pb.beam_select(v, 4, 8, cum=cum)] for v in x]
    graphs, outs = [], []
    for v in x:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(pb.beam_select(v, 4, 8, cum=cum))
        graphs.append(g)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for g, st in zip(graphs, s):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))


def test_empty_batch():
    x = torch.zeros(0, 100, device="cuda")
    s, t, p = pb.beam_select(x, 4, 8)
    assert s.shape == (0, 8) and t.shape == (0, 8) and p.shape == (0, 8)
    pb.beam_reorder(torch.zeros(0, 3, device="cuda"), torch.zeros(0, 4, dtype=torch.int32, device="cuda"))
