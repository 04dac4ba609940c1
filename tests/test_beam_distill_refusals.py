"""What the beam search and distillation entry points refuse, before any device
work (no GPU needed), and the host-side layout of reordered states."""
import ctypes

import numpy as np
import pytest
import torch

import pesti_beam as pb
import pesti_distill as pd
import pesti_sampler as ps

BAD = ps.PESTI_E_INVALID_ARG
P = 1 << 20  # an address that is never used: every call below is refused first


@pytest.fixture(scope="module")
def lib():
    return ps.load_library()


SELECT = dict(logits=P, dtype=ps.PESTI_F32, G=2, W=4, V=100, ld=100, cum=None, done=None, K=8, score=P, token=P,
              parent=P, lse=None, ws=P, ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change,msg", [
    (dict(dtype=ps.PESTI_FP8_E4M3), "f32, bf16 or f16"), (dict(G=-1), "G < 0"), (dict(W=0), "W must"),
    (dict(W=65), "W must"), (dict(K=0), "K must"), (dict(K=129), "K must"), (dict(V=0), "V must"),
    (dict(V=1 << 31, ld=1 << 31), "V must"), (dict(ld=99), "ld is below"), (dict(logits=None), "null logits"),
    (dict(score=None), "null output"), (dict(token=None), "null output"), (dict(parent=None), "null output"),
    (dict(logits=P + 2), "not aligned"), (dict(ws=None), "workspace too small"), (dict(ws_bytes=100), "workspace too"),
    (dict(ws=P + 16), "256-byte"), (dict(G=1 << 40), "too large"),
])
def test_select_refusals(lib, change, msg):
    assert lib.pesti_beam_select(*{**SELECT, **change}.values()) == BAD
    assert msg in lib.pesti_last_error().decode()


def test_select_workspace(lib):
    small = lib.pesti_beam_select_workspace(ps.PESTI_BF16, 1, 4, 1000, 8)
    assert 0 < small < lib.pesti_beam_select_workspace(ps.PESTI_F32, 1, 4, 128256, 8)
    assert lib.pesti_beam_select_workspace(ps.PESTI_BF16, 1, 65, 1000, 8) == BAD
    assert lib.pesti_beam_select(*{**SELECT, "G": 0}.values()) == ps.PESTI_OK  # nothing to do


def _state(**change):
    s = pb._StateC(*[P] * 10, 16)
    for k, v in change.items():
        setattr(s, k, v)
    return s


def _advance(lib, state=None, score=P, token=P, parent=P, G=2, W=4, K=8, stop=P, n_stop=1, limits=None):
    state = state if state is not None else _state()
    limits = limits if limits is not None else pb._LimitsC(16, 16, 1.0, 0)
    return lib.pesti_beam_advance(ctypes.addressof(state), score, token, parent, G, W, K, stop, n_stop,
                                  ctypes.addressof(limits), None)


@pytest.mark.parametrize("change", [
    dict(G=-1), dict(W=0), dict(W=65), dict(K=0), dict(K=129), dict(n_stop=-1), dict(score=None), dict(token=None),
    dict(parent=None), dict(stop=None), dict(state=_state(cum=None)), dict(state=_state(done=None)),
    dict(state=_state(fin_tokens=None)), dict(state=_state(cap=-1)), dict(state=_state(cap=8)),
    dict(limits=pb._LimitsC(-1, 16, 1.0, 0)), dict(limits=pb._LimitsC(16, -1, 1.0, 0)),
    dict(limits=pb._LimitsC(1 << 31, 1 << 31, 1.0, 0)), dict(limits=pb._LimitsC(16, 16, float("nan"), 0)),
])
def test_advance_refusals(lib, change):
    assert _advance(lib, **change) == BAD
    assert lib.pesti_last_error()


def test_reset_refusals(lib):
    s = _state(tokens=None)
    assert lib.pesti_beam_reset(ctypes.addressof(s), 2, 4, None) == BAD
    assert lib.pesti_beam_reset(None, 2, 4, None) == BAD
    ok = _state()
    assert lib.pesti_beam_reset(ctypes.addressof(ok), 2, 65, None) == BAD
    assert lib.pesti_beam_reset(ctypes.addressof(ok), 0, 4, None) == ps.PESTI_OK


def _reorder(lib, rows, parent=P, G=2, W=4, n=None):
    arr = (pb._RowsC * max(1, len(rows)))(*rows)
    return lib.pesti_beam_reorder(ctypes.addressof(arr), len(rows) if n is None else n, parent, G, W, None)


def _rows(src=P, dst=P, src_row=64, dst_row=64, src_blk=0, dst_blk=0, blocks=1, nbytes=64):
    return pb._RowsC(src, dst, src_row, dst_row, src_blk, dst_blk, blocks, nbytes)


@pytest.mark.parametrize("rows,more", [
    ([_rows(src=None)], {}), ([_rows(dst=None)], {}), ([_rows()], dict(parent=None)), ([_rows()], dict(W=0)),
    ([_rows()], dict(W=65)), ([_rows()], dict(G=-1)), ([_rows()], dict(n=-1)),
    ([_rows(src_row=-64)], {}), ([_rows(blocks=-1)], {}), ([_rows(nbytes=-1)], {}),
    ([_rows(dst=P + 64)], {}),                                    # partial overlap
    ([_rows(dst=P - 1)], {}),
    ([_rows(src_row=128)], {}),                                   # in place with unequal strides
    ([_rows(dst=2 * P, dst_row=32)], {}),                         # rows that overlap
    ([_rows(dst=2 * P, blocks=2, dst_blk=32, dst_row=256)], {}),  # blocks that overlap
    ([_rows(dst=2 * P, blocks=2, dst_blk=100, dst_row=70, src_blk=100)], {}),  # interleaved rows
    ([_rows(), _rows()], {}),                                     # the same state twice
    ([_rows(src=2 * P), _rows()], {}),
])
def test_reorder_refusals(lib, rows, more):
    assert _reorder(lib, rows, **more) == BAD
    assert lib.pesti_last_error()


def test_reorder_refuses_before_it_launches(lib):
    # a state of more tiles than a grid has, behind one that could be moved
    large = _rows(src=2 * P, dst=2 * P, src_row=1, dst_row=1, src_blk=8, dst_blk=8, blocks=1 << 31, nbytes=1)
    assert _reorder(lib, [_rows(), large]) == BAD
    assert "too large" in lib.pesti_last_error().decode()


def test_reorder_of_nothing(lib):
    assert _reorder(lib, [], parent=None) == ps.PESTI_OK
    assert _reorder(lib, [_rows()], parent=None, G=0) == ps.PESTI_OK


DISTILL = dict(logits=P, dtype=ps.PESTI_F32, N=4, V=100, ld=100, idx=P, idx_ld=8, val=P, vtype=ps.PESTI_F32, val_ld=8,
               k=8, lse=None, weight=None, T=1.0)
COMMON = [
    (dict(dtype=ps.PESTI_FP8_E5M2), "logits must be"), (dict(vtype=ps.PESTI_FP8_E4M3), "teacher values"),
    (dict(N=-1), "N < 0"), (dict(V=0), "V must"), (dict(V=1 << 31, ld=1 << 31), "V must"), (dict(ld=99), "ld is below"),
    (dict(k=0), "k must"), (dict(k=257), "k must"), (dict(idx_ld=-1), "negative stride"),
    (dict(val_ld=-8), "negative stride"), (dict(T=0.0), "temperature"), (dict(T=float("nan")), "temperature"),
    (dict(T=-1.0), "temperature"), (dict(T=float("inf")), "temperature"), (dict(T=1e-4), "temperature"),
    (dict(logits=None), "null"), (dict(idx=None), "null"), (dict(val=None), "null"), (dict(logits=P + 1), "not aligned"),
    (dict(val=P + 2), "teacher values are not aligned"), (dict(vtype=ps.PESTI_BF16, val=P + 1), "teacher values are not"),
]


@pytest.mark.parametrize("change,msg", COMMON)
def test_distill_common_refusals(lib, change, msg):
    a = list({**DISTILL, **change}.values())
    assert lib.pesti_distill_topk(*a, P, None, None, 0, P, 1 << 30, None) == BAD
    assert msg in lib.pesti_last_error().decode()
    assert lib.pesti_distill_topk_backward(*a, P, P, 1, 2 * P, 100, None) == BAD
    assert msg in lib.pesti_last_error().decode()


def test_distill_output_refusals(lib):
    a = list(DISTILL.values())
    b = lib.pesti_distill_topk_backward

    def f(*args):
        return lib.pesti_distill_topk(*args[:-1], P, 1 << 30, args[-1])

    assert f(*a, None, None, None, 0, None) == BAD                     # no loss
    assert f(*a, P, None, 2 * P, 99, None) == BAD                      # grad_ld
    assert f(*a, P, None, 2 * P + 2, 100, None) == BAD                 # alignment
    assert f(*a, P, None, P + 4, 100, None) == BAD                     # overlap that is not in place
    assert f(*a, P, None, P, 101, None) == BAD                         # in place with another stride
    assert f(*a, P, 3 * P, P, 100, None) == BAD                        # in place, but the logits are needed again
    assert b(*a, None, P, 1, 2 * P, 100, None) == BAD
    assert b(*a, P, None, 1, 2 * P, 100, None) == BAD
    assert b(*a, P, P, 1, None, 100, None) == BAD
    assert b(*a, P, P, -1, 2 * P, 100, None) == BAD
    assert f(*list({**DISTILL, "N": 0}.values()), None, None, None, 0, None) == ps.PESTI_OK
    for ws, size in ((None, 1 << 30), (P, 64), (P + 8, 1 << 30)):
        assert lib.pesti_distill_topk(*a, P, None, None, 0, ws, size, None) == BAD
        assert "workspace" in lib.pesti_last_error().decode()
    need = lib.pesti_distill_topk_workspace
    assert 0 < need(ps.PESTI_BF16, 4, 1000, 8) < need(ps.PESTI_F32, 40, 100000, 256)
    for bad in ((ps.PESTI_FP8_E4M3, 4, 100, 8), (0, -1, 100, 8), (0, 4, 0, 8), (0, 4, 100, 257), (0, 1 << 40, 100, 8)):
        assert need(*bad) == BAD


def test_python_checks():
    x = torch.zeros(4, 10)
    with pytest.raises(ValueError, match="CUDA"):
        pb.beam_select(x, 2, 4)
    with pytest.raises(ValueError, match="multiple"):
        pb.beam_select(x, 3, 4)
    with pytest.raises(ValueError, match="float32, bfloat16"):
        pb.beam_select(x.double(), 2, 4)
    with pytest.raises(ValueError, match="contiguous"):
        pb.beam_select(torch.zeros(10, 4).t(), 2, 4)
    with pytest.raises(ValueError, match="cum"):
        pb.beam_select(x, 2, 4, cum=torch.zeros(4, dtype=torch.float64))
    with pytest.raises(ValueError, match="k must"):
        pb.beam_select(x, 2, 129)
    idx, val = torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, 3)
    with pytest.raises(ValueError, match="CUDA"):
        pd.distill_topk(x, idx, val)
    with pytest.raises(ValueError, match="int32"):
        pd.distill_topk(x, idx.long(), val)
    with pytest.raises(ValueError, match="same shape"):
        pd.distill_topk(x, idx, val[:, :2])
    with pytest.raises(ValueError, match="weight"):
        pd.distill_topk(x, idx, val, weight=torch.ones(4, 1))
    with pytest.raises(ValueError, match="first dimension"):
        pb.beam_reorder(torch.zeros(5, 3), torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="parent"):
        pb.beam_reorder(torch.zeros(4, 3), torch.zeros(2, 2, dtype=torch.int64))


@pytest.mark.parametrize("make,want", [
    (lambda: torch.zeros(6, 4), (1, 4, 0)),
    (lambda: torch.zeros(6), (1, 1, 0)),
    (lambda: torch.zeros(6, 4, 8, 2)[:, :, :5], (4, 10, 16)),
    (lambda: torch.zeros(6, 4, 8, 2)[:, 1:3, :5], (2, 10, 16)),
    (lambda: torch.zeros(6, 2, 3, 8)[..., :5], (6, 5, 8)),
    (lambda: torch.zeros(6, 1, 8), (1, 8, 0)),
    (lambda: torch.zeros(6, 3, 8)[:, ::2], (2, 8, 16)),
])
def test_row_blocks(make, want):
    t = make()
    assert pb._layout(t.shape, t.stride()) == want


def test_row_blocks_refuses_two_strides():
    with pytest.raises(ValueError):
        t = torch.zeros(6, 4, 5, 8)[:, :3, :4, :2]
        pb._layout(t.shape, t.stride())


def test_oracle_against_a_direct_search():
    """The oracle's selection against every (beam, token) pair sorted."""
    import beam as OB
    rng = np.random.default_rng(3)
    x = rng.normal(size=(6, 40)).astype(np.float32)
    cum = rng.normal(size=(2, 3)).astype(np.float32)
    score, token, parent, _ = OB.select(x, 3, 7, cum)
    for g in range(2):
        every = []
        for w in range(3):
            z = x[g * 3 + w].astype(np.float64)
            lp = z - np.log(np.exp(z).sum())
            every += [(-(float(cum[g, w]) + lp[v]), w, v) for v in range(40)]
        every.sort()
        assert [(w, v) for _, w, v in every[:7]] == list(zip(parent[g], token[g]))
        assert np.allclose([-e[0] for e in every[:7]], score[g], atol=1e-12)


def test_oracle_gradient_against_differences():
    """The oracle's gradient against central differences of its loss."""
    import distill as OD
    rng = np.random.default_rng(4)
    x = rng.normal(size=20) * 2
    idx = np.array([3, 7, 3, -1, 19, 40])
    val = rng.normal(size=6)
    for lse in (None, 3.0):
        _, grad, *_ = OD.row(x, idx, val, 1.5, lse, 0.7)
        h = 1e-5
        for v in range(20):
            d = np.zeros(20)
            d[v] = h
            up, dn = OD.row(x + d, idx, val, 1.5, lse, 0.7)[0], OD.row(x - d, idx, val, 1.5, lse, 0.7)[0]
            # central differences: h^2/6 times a third derivative of order 1, and 1e-16/h of rounding
            assert abs((up - dn) / (2 * h) - grad[v]) < 1e-9
