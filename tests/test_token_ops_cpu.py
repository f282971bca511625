"""Argument checks of the linear layer and the root-mean-square norm (no GPU: the records are only validated)."""
import pytest

from denox_b200 import lib

X, R, W, S, O, SC = (0x10000000 * i for i in range(1, 7))  # far apart; never read


def norm(**kw):
    a = dict(rows=4, channels=64, x=X, out=O, residual=R, weight=W, sum_out=S)
    a.update(kw)
    return lib.L.dnxcu_rmsnorm_validate(lib.rmsnorm_desc(**a))


def test_rmsnorm_accepts():
    assert norm() == lib.OK
    assert norm(residual=None, weight=None, sum_out=None) == lib.OK
    assert norm(out_dtype=lib.DT_E4M3, out_scale=SC) == lib.OK
    assert norm(sum_out=R) == lib.OK and norm(sum_out=X, out=R) == lib.OK  # in place
    assert norm(rows=1, channels=1) == lib.OK
    # windows side by side in the same wider rows
    assert norm(x=X, x_stride=256, out=X + 2 * 64, out_stride=256, residual=X + 2 * 192, residual_stride=256) == lib.OK


@pytest.mark.parametrize("kw", [dict(rows=0), dict(rows=-1), dict(channels=0), dict(x=None), dict(out=None), dict(out_dtype=2),
                                dict(out_dtype=lib.DT_E4M3), dict(out_scale=SC), dict(eps=0.0), dict(eps=-1.0),
                                dict(eps=float("nan")), dict(eps=float("inf")), dict(x_stride=63), dict(residual_stride=-64),
                                dict(sum_stride=1), dict(out_stride=32)])
def test_rmsnorm_bad_arguments(kw):
    assert norm(**kw) == lib.E_BAD_ARG


@pytest.mark.parametrize("kw", [dict(x=X + 1), dict(out=O + 1), dict(residual=R + 1), dict(weight=W + 1), dict(sum_out=S + 1),
                                dict(out_dtype=lib.DT_E4M3, out_scale=SC + 2)])
def test_rmsnorm_misaligned(kw):
    assert norm(**kw) == lib.E_MISALIGNED


@pytest.mark.parametrize("kw", [dict(rows=1 << 31), dict(channels=(1 << 24) + 1), dict(x_stride=1 << 35)])
def test_rmsnorm_limits(kw):
    assert norm(**kw) == lib.E_LIMIT


@pytest.mark.parametrize("kw", [dict(out=X + 2), dict(out=S), dict(sum_out=X + 128), dict(out=W), dict(sum_out=W),
                                dict(out=X, out_stride=128), dict(out_dtype=lib.DT_E4M3, out=X, out_scale=SC),
                                dict(out_dtype=lib.DT_E4M3, out_scale=O), dict(out_dtype=lib.DT_E4M3, out_scale=X),
                                dict(x=X, x_stride=256, out=X + 2 * 224, out_stride=256)])
def test_rmsnorm_overlap(kw):
    """An output that shares bytes with another operand, other than exactly in place."""
    assert norm(**kw) == lib.E_BAD_ARG
