"""Beam selection where teams of fewer warps take the beams, and over rows of so
many columns that a key stands for a run of segments, against the 64-bit oracle
(oracle/beam.py).  Tolerances are test_beam_gpu.py's."""
import numpy as np
import pytest
import torch

import beam as OB
import pesti_beam as pb
from test_beam_gpu import DT, NEG, _check
from test_beam_plan import plan

pytestmark = pytest.mark.gpu

CODE = {"f32": pb.PESTI_F32, "bf16": pb.PESTI_BF16, "f16": pb.PESTI_F16}


def _plan(dtype, G, W, V, K):
    return plan(CODE[dtype], G, W, V, K, torch.cuda.get_device_properties(0).multi_processor_count)


def _want(rows, W, K, cum):
    """oracle.beam.select, which sorts whole rows, on what can be among a row's K largest."""
    G, V = rows.shape[0] // W, rows.shape[1]
    score, token, parent = np.full((G, K), NEG), np.full((G, K), -1), np.full((G, K), -1)
    for g in range(G):
        have = []
        for w in range(W):
            row = rows[g * W + w]
            logp, _ = OB.row_logp(row)
            at = np.nonzero((row >= np.partition(row, V - K)[V - K]) & (row > NEG))[0]
            at = at[np.lexsort((at, -row[at].astype(np.float64)))][:K]
            have += [(-(float(cum[g, w]) + logp[v]), w, r, v) for r, v in enumerate(at)]
        have.sort()
        for r, (neg, w, _, v) in enumerate(have[:K]):
            score[g, r], token[g, r], parent[g, r] = -neg, v, w
    return score, token, parent


def _check_live(x, live, W, K, cum):
    """beam_select of a batch of which only the groups `live` are running: nothing of the others is read."""
    G = x.shape[0] // W
    done = torch.ones(G, dtype=torch.uint8, device="cuda")
    done[live] = 0
    rows = torch.cat([x[g * W:(g + 1) * W] for g in live]).float().cpu().numpy()
    want = _want(rows, W, K, cum[live].cpu().numpy())
    s, t, p = pb.beam_select(x, W, K, cum=cum, done=done)
    assert np.array_equal(t[live].cpu().numpy(), want[1]) and np.array_equal(p[live].cpu().numpy(), want[2])
    got = s[live].cpu().numpy().astype(np.float64)
    fine = want[2] >= 0
    assert np.all(got[~fine] == NEG)
    assert np.all(np.abs(got[fine] - want[0][fine]) <= 3e-6 + np.abs(want[0][fine]) * 2.0 ** -24)
    rest = done.bool()
    assert torch.isneginf(s[rest]).all() and (t[rest] == -1).all() and (p[rest] == -1).all()


def _fill(row, kind):
    if kind == "random":
        row.normal_(0, 3)
    elif kind == "steps":      # hundreds of segments share the K-th largest maximum
        row.normal_(0, 1).round_()
    elif kind == "few":        # fewer finite segments than candidates
        row.fill_(NEG)
        row[17::row.numel() // 9] = torch.arange(len(range(17, row.numel(), row.numel() // 9))).to(row)
    elif kind == "rising":     # all candidates in the last segments
        row.copy_(torch.arange(row.numel(), device=row.device).div(row.numel() / 200).to(row.dtype))
    elif kind == "none":
        row.fill_(NEG)


@pytest.mark.parametrize("dtype,V,W,K,run", [
    ("f32", 4_000_003, 2, 16, 2), ("f32", 5_401_162, 2, 16, 3), ("bf16", 10_900_007, 2, 128, 3),
    ("f16", 10_900_007, 2, 8, 3), ("f32", 12_101_363, 1, 8, 3),
])
def test_runs_of_segments(dtype, V, W, K, run):
    p = _plan(dtype, 1, W, V, K)
    assert p["run"] == run and p["team_warps"] == 7
    torch.manual_seed(V)
    x = torch.empty(W, V, dtype=DT[dtype], device="cuda")
    cum = torch.linspace(0.0, -0.5, W).view(1, W).cuda()
    for kinds in (("random", "random"), ("steps", "few"), ("rising", "none")):
        for row, kind in zip(x, kinds):
            _fill(row, kind)
        _check_live(x, [0], W, K, cum)


@pytest.mark.parametrize("dtype,G,W,V,K,run,team", [
    ("f32", 44, 8, 2_700_001, 16, 3, 3), ("f32", 80, 8, 1_300_001, 16, 3, 1), ("bf16", 80, 8, 2_600_003, 40, 2, 3),
])
def test_runs_of_segments_in_large_batches(dtype, G, W, V, K, run, team):
    p = _plan(dtype, G, W, V, K)
    assert p["run"] == run and p["team_warps"] == team
    torch.manual_seed(G)
    x = torch.empty(G * W, V, dtype=DT[dtype], device="cuda")
    live = [0, G - 1]
    for g in live:
        for row, kind in zip(x[g * W:], ("random", "steps", "few", "none", "rising", "random", "steps", "random")):
            _fill(row, kind)
    cum = -torch.rand(G, W, device="cuda")
    _check_live(x, live, W, K, cum)


def _batch(rows, G):
    """G groups of the same rows, each group's turned by one beam more."""
    return torch.cat([rows.roll(g, 0) for g in range(G)])


# W, G, K and the warps of a team; the cluster's blocks do not stay
TEAMS = [(10, 40, 20, 3), (10, 60, 20, 1), (10, 60, 64, 3), (3, 250, 6, 1), (16, 30, 128, 3)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("W,G,K,team", TEAMS)
def test_masks_in_large_batches(dtype, W, G, K, team):
    V = 5003
    p = _plan(dtype, G, W, V, K)
    assert p["team_warps"] == team and p["stay"] == 0
    x = torch.randn(W, V, generator=torch.Generator().manual_seed(W)).mul(3.0).to(DT[dtype]).cuda()
    x[0] = NEG
    x[1] = NEG
    x[1, 4711] = -2.0
    x[2] = NEG
    x[2, 17::1001] = torch.arange(len(range(17, V, 1001))).to(x.dtype).cuda()
    if W > 3:
        x[3, ::3] = float("nan")
        x[4, 99] = x[4, 4000] = float("inf")
        x[5] = torch.finfo(x.dtype).min
        x[6, 1:] = torch.finfo(x.dtype).min
        x[7] = float("nan")
    cum = -torch.rand(G, W, generator=torch.Generator().manual_seed(G)).cuda()
    cum[::3, 1] = NEG
    cum[::5, 2] = float("nan")
    done = torch.arange(G).cuda() % 11 == 7
    _check(_batch(x, G), W, K, cum, done)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("W,G,K,team", TEAMS)
def test_ties_in_large_batches(dtype, W, G, K, team):
    """Rows of few values, so that a list is filled in rounds and more candidates are equal than are ranked."""
    V = 3001
    p = _plan(dtype, G, W, V, K)
    assert p["team_warps"] == team and p["stay"] == 0
    at = torch.arange(V).cuda()
    x = torch.zeros(W, V, dtype=DT[dtype], device="cuda")
    x[1] = at.div(3, rounding_mode="floor").neg().to(x.dtype)
    x[2] = (at % 3).to(x.dtype)
    if W > 3:
        x[3] = at.to(x.dtype)
        x[4] = 7.0
        x[5, 2000:] = 1.0
        x[6, ::2] = -0.0
    _check(_batch(x, G), W, K)
    cum = -0.5 * (torch.arange(G * W).view(G, W) % 2).float().cuda()
    _check(_batch(x, G), W, K, cum)


@pytest.mark.parametrize("shift", [0.0, 1e-7, 4e-7, 2e-6])
@pytest.mark.parametrize("W,G,K,team,blocks", [(6, 60, 24, 3, 2), (8, 80, 24, 1, 1), (12, 40, 40, 3, 3)])
def test_near_ties_in_large_batches(shift, W, G, K, team, blocks):
    """Equal rows with scores a few f32 steps apart, at different alignments: one block adds the rows up again."""
    V = 9011
    p = _plan("f32", G, W, V, K)
    assert p["team_warps"] == team and p["blocks"] == blocks and p["stay"] == 0
    buf = torch.zeros(G * W, V + 2).cuda()
    buf[:, :V] = torch.randn(V, generator=torch.Generator().manual_seed(V)).mul(3.0).cuda()
    order = [torch.randperm(W, generator=torch.Generator().manual_seed(g)) for g in range(G)]
    cum = (torch.stack(order) * shift).cuda()
    _check(buf[:, :V], W, K, cum)
