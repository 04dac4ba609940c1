"""The layout of the beam selection's second kernel, computed on the host for
every size that the call takes (no GPU needed)."""
import ctypes
import random

import pytest

import pesti_sampler as ps

FIELDS = ("segments", "team_warps", "teams", "blocks", "stay", "run", "keys", "team_at", "team_stride", "keys_at",
          "hist_at", "bytes", "most_bytes")
SMS = 148


def plan(dtype, G, W, V, K, sms=SMS):
    out = (ctypes.c_int64 * len(FIELDS))()
    assert ps.load_library().pesti_testing_beam_plan(dtype, G, W, V, K, sms, ctypes.addressof(out)) == ps.PESTI_OK
    return dict(zip(FIELDS, out))


def _holds(p, W, K):
    # 16-byte reads: the keys as they are copied, the histogram as it is searched
    assert p["team_at"] % 16 == 0 and p["team_stride"] % 16 == 0 and p["keys_at"] % 16 == 0 and p["hist_at"] % 16 == 0
    # a key for every segment, and the words behind the keys
    assert p["keys"] * p["run"] >= p["segments"]
    assert p["run"] > 1 or p["keys"] == p["segments"]
    assert p["hist_at"] >= p["keys_at"] + 4 * p["keys"]
    # the histogram, the selected segments and 32 words behind it
    assert p["team_stride"] >= p["hist_at"] + 4 * (256 + (128 + 64 + 8) + 32)
    # the teams' arrays, and the merge's scores in their place
    assert p["bytes"] >= p["team_at"] + max(p["teams"] * p["team_stride"], 8 * W * K)
    assert p["bytes"] <= p["most_bytes"] == 200 * 1024
    assert 1 <= p["blocks"] <= 8 and 1 <= p["teams"] * (p["team_warps"] + 1) <= 16


# rows that do not fit a key per segment, by hand: groups, beams, columns, candidates, segments of a key
LONG = [
    (ps.PESTI_F32, 1, 1, 12_101_363, 8, 3), (ps.PESTI_F32, 1, 2, 5_401_162, 16, 3),
    (ps.PESTI_F32, 1, 2, 4_000_003, 16, 2), (ps.PESTI_F32, 40, 64, 1_601_048, 128, 3), (ps.PESTI_F32, 80, 8, 1_300_001, 16, 3),
    (ps.PESTI_F32, 40, 8, 2_700_001, 16, 3), (ps.PESTI_BF16, 1, 4, 10_900_007, 8, 3),
]


@pytest.mark.parametrize("dtype,G,W,V,K,run", LONG)
def test_long_rows(dtype, G, W, V, K, run):
    p = plan(dtype, G, W, V, K)
    assert p["run"] == run
    _holds(p, W, K)


@pytest.mark.parametrize("dtype", [ps.PESTI_F32, ps.PESTI_BF16])
def test_every_width(dtype):
    for W in range(1, 65):
        for G in (1, 20, 40, 200):
            for K in (1, 2, 31, 33, 127, 128):
                for V in (1, 4097, 256_000, 2_700_001, 12_101_363, 2**31 - 1):
                    if G * W * (V // (2048 if dtype == ps.PESTI_BF16 else 1024) + 5) > 2**31:
                        continue
                    _holds(plan(dtype, G, W, V, K), W, K)


def test_drawn_sizes():
    rng = random.Random(7)
    runs = set()
    for _ in range(20000):
        W, K = rng.randint(1, 64), rng.randint(1, 128)
        V = int(2 ** rng.uniform(0, 28))
        G = int(2 ** rng.uniform(0, 8))
        p = plan(rng.choice([ps.PESTI_F32, ps.PESTI_BF16, ps.PESTI_F16]), G, W, V, K, rng.choice([SMS, 132, 20]))
        _holds(p, W, K)
        runs.add(min(p["run"], 5))
    assert runs == {1, 2, 3, 4, 5}
