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


XS, WS = 0x70000000, 0x80000000
ST = 0x90000000


def linear(**kw):
    a = dict(rows=40, c_in=64, c_out=96, x=X, weights=W, out=O, residual=R, bias=S, x_scale=XS, w_scale=WS)
    a.update(kw)
    return lib.linear_desc(**a)


def test_linear_accepts_and_picks():
    def pick(**kw):
        d = linear(**kw)
        st = lib.L.dnxcu_linear_validate(d)
        got = lib.L.dnxcu_linear_pick(d)
        assert (st == lib.OK) == (got > 0) and (st == lib.OK or st == got)
        return got

    assert pick(rows=1) == lib.LINEAR_ROWS
    assert pick(rows=100, c_in=4096, c_out=4096) == lib.LINEAR_SPLIT and pick(rows=100) == lib.LINEAR_TILE
    assert pick(rows=300, c_in=16384, c_out=1024) == lib.LINEAR_SPLIT and pick(rows=300, c_in=512, c_out=8192) == lib.LINEAR_TILE
    assert pick(rows=100000) == lib.LINEAR_TILE
    assert pick(rows=100000, dtype=lib.DT_E4M3) == lib.LINEAR_TILE
    assert pick(c_in=65) == lib.LINEAR_ANY and pick(x=X + 2) == lib.LINEAR_ANY and pick(weights=W + 8) == lib.LINEAR_ANY
    assert pick(c_in=65, x_stride=72, w_stride=80) != lib.LINEAR_ANY  # padded rows
    assert pick(dtype=lib.DT_E4M3, c_in=72) == lib.LINEAR_ANY
    # thin layers over many packed rows: several at a time, whatever the alignment of a single one
    thin = dict(rows=522240, c_in=9, c_out=32, x_scale=None, residual=None, out=0x100000000)
    assert pick(**thin) == lib.LINEAR_TILE
    for kw in (dict(x_stride=10), dict(out_stride=40), dict(x_scale=XS), dict(rows=1000), dict(x=X + 2), dict(c_out=40)):
        assert pick(**{**thin, **kw}) == lib.LINEAR_ANY
    assert pick(residual=None, bias=None, x_scale=None, w_scale=None, rows=1, c_in=1, c_out=1) == lib.LINEAR_ANY
    assert pick(residual=O) > 0  # in place
    for v, kw in ((lib.LINEAR_ROWS, dict(rows=16)), (lib.LINEAR_SPLIT, {}), (lib.LINEAR_TILE, {}), (lib.LINEAR_ANY, {})):
        assert pick(variant=v, **kw) == v
    for v, kw in ((lib.LINEAR_ROWS, dict(rows=17)), (lib.LINEAR_ROWS, dict(rows=4, c_in=68, x_stride=72, w_stride=72)),
                  (lib.LINEAR_SPLIT, dict(x=X + 2)), (lib.LINEAR_TILE, dict(c_in=65))):
        assert pick(variant=v, **kw) == lib.E_UNSUPPORTED


@pytest.mark.parametrize("kw", [dict(rows=0), dict(c_in=0), dict(c_out=-5), dict(x=None), dict(weights=None), dict(out=None),
                                dict(dtype=2), dict(dtype=-1), dict(activation=6), dict(activation=-1), dict(variant=5),
                                dict(x_stride=63), dict(w_stride=1), dict(out_stride=95), dict(residual_stride=-96)])
def test_linear_bad_arguments(kw):
    assert lib.L.dnxcu_linear_validate(linear(**kw)) == lib.E_BAD_ARG


@pytest.mark.parametrize("kw", [dict(x=X + 1), dict(weights=W + 1), dict(out=O + 1), dict(residual=R + 1), dict(bias=S + 1),
                                dict(x_scale=XS + 2), dict(w_scale=WS + 1), dict(device_status=ST + 1)])
def test_linear_misaligned(kw):
    assert lib.L.dnxcu_linear_validate(linear(**kw)) == lib.E_MISALIGNED


@pytest.mark.parametrize("kw", [dict(rows=1 << 31), dict(c_in=(1 << 24) + 1), dict(c_out=(1 << 24) + 1), dict(x_stride=1 << 35),
                                dict(out_stride=1 << 35)])
def test_linear_limits(kw):
    assert lib.L.dnxcu_linear_validate(linear(**kw)) == lib.E_LIMIT


@pytest.mark.parametrize("kw", [dict(out=X), dict(out=W), dict(out=R + 2), dict(residual=O, residual_stride=128), dict(bias=O),
                                dict(x_scale=O + 4), dict(w_scale=O), dict(device_status=O), dict(out=X + 64 * 39 * 2)])
def test_linear_overlap(kw):
    assert lib.L.dnxcu_linear_validate(linear(**kw)) == lib.E_BAD_ARG


def test_null_records():
    import ctypes as C
    p = C.c_void_p()
    assert lib.L.dnxcu_linear_validate(None) == lib.E_BAD_ARG and lib.L.dnxcu_linear_launch(None, None) == lib.E_BAD_ARG
    assert lib.L.dnxcu_linear_plan_create(None, C.byref(p)) == lib.E_BAD_ARG
    assert lib.L.dnxcu_linear_plan_create(linear(), None) == lib.E_BAD_ARG
    assert lib.L.dnxcu_linear_plan_launch(None, None) == lib.E_BAD_ARG
    assert lib.L.dnxcu_rmsnorm_validate(None) == lib.E_BAD_ARG and lib.L.dnxcu_rmsnorm_launch(None, None) == lib.E_BAD_ARG
    lib.L.dnxcu_linear_plan_destroy(None)
