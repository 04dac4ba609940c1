"""What the cross entropy's entry points that pass on each row's -log p refuse, before any device work (no GPU needed)."""
import pytest

import pesti_sampler as ps
import test_head_refusals as R


@pytest.fixture(scope="module")
def lib():
    return ps.load_library()


def _with_nll(args, nll):
    at = list(args).index("lse") + 1
    items = list(args.items())
    return dict(items[:at] + [("nll", nll)] + items[at:])


@pytest.mark.parametrize("change,msg", R.COMMON + [(dict(nll=R.P + 2), "loss or lse is not"), (dict(loss=None), "null loss")])
def test_forward(lib, change, msg):
    args = {**R.CE, **_with_nll(R.FORWARD, R.P)}
    assert lib.pesti_linear_ce_nll(*{**args, **change}.values()) == R.BAD
    assert msg in lib.pesti_last_error().decode()
    assert lib.pesti_linear_ce_nll(*{**args, "N": 0}.values()) == ps.PESTI_OK


@pytest.mark.parametrize("change,msg", R.COMMON + [
    (dict(nll=R.P + 1), "gradient is not aligned"), (dict(lse=None), "null lse"), (dict(up=None), "null lse"),
])
def test_backward(lib, change, msg):
    args = {**R.CE, **_with_nll(R.BACKWARD, R.P)}
    assert lib.pesti_linear_ce_nll_backward(*{**args, **change}.values()) == R.BAD
    assert msg in lib.pesti_last_error().decode()
    assert lib.pesti_linear_ce_nll_backward(*{**args, "N": 0, "gw": None}.values()) == ps.PESTI_OK


def test_giving_up(lib):
    for product, round in ((-1, 0), (5, 0), (0, -2)):
        assert lib.pesti_testing_give_up(product, round) == R.BAD
    assert lib.pesti_testing_give_up(4, -1) == ps.PESTI_OK
