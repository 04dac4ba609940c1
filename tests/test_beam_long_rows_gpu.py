"""Beam selection where teams of fewer warps take the beams, and over rows of so
many columns that a key stands for a run of segments, against the 64-bit oracle
(oracle/beam.py).  Tolerances are test_beam_gpu.py's."""
import numpy as np
import pytest
import torch

import beam as OB
import pesti_beam as pb
from test_beam_gpu import DT, NEG
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
