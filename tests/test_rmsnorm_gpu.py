"""Root-mean-square norm on the GPU against its formula in 64 bits.

Tolerances.  Sums and statistics are 32 bit: a sum of squares of n terms that a thread adds one after the other and
warps join as a tree is off by at most (n_seq + 12) 2^-24 relative, its root by half of that; at the sizes below
n_seq <= 70, so with the few further roundings y is within 2^-18 of itself before the output's rounding.  The output's
rounding adds half a step: 2^-11 |y| in binary16 (2^-25 below its normal range), 2^-4 |y| in e4m3 (2^-10 below 2^-6)."""
import pytest
import torch

from denox_b200 import lib
from token_util import Mat, assert_within, normal

pytestmark = pytest.mark.gpu
EPS = 1e-5


def reference(x, residual, weight, eps=EPS):
    h = x.double() if residual is None else x.double() + residual.double()
    w = 1.0 if weight is None else weight.double()
    return h, w * h / torch.sqrt((h * h).mean(1, keepdim=True) + eps)


def tol_f16(v):
    return v.abs() * (2.0 ** -11 + 2.0 ** -18) + 2.0 ** -25


def tol_e4m3(v):
    return v.abs() * (2.0 ** -4 + 2.0 ** -18) + 2.0 ** -10


def check_out(out, scale, y):
    if scale is None:
        assert_within(out, y, tol_f16(y), "out")
        return
    top = y.abs().amax(1)
    s = torch.where(top > 0, top / 448.0, torch.ones_like(top))
    assert_within(scale, s, s * 2.0 ** -18, "scale")
    v = y / s[:, None]
    assert_within(out, v, tol_e4m3(v), "out")


def run(x, residual=None, weight=None, q=False, keep_sum=False, eps=EPS, strides=(0, 0, 0, 0), offsets=(0, 0, 0, 0), stream=0):
    """Launches the norm on guarded copies; returns (out, scale, sum) on the host."""
    rows, c = x.shape
    pick = lambda i: dict(stride=strides[i] or None, offset=offsets[i])
    mx = Mat(rows, c, data=x, **pick(0))
    mr = Mat(rows, c, data=residual, **pick(1)) if residual is not None else None
    mw = Mat(1, c, data=weight[None], offset=offsets[0]) if weight is not None else None
    ms = Mat(rows, c, **pick(2)) if keep_sum else None
    mo = Mat(rows, c, torch.float8_e4m3fn if q else torch.float16, **pick(3))
    msc = Mat(1, rows, torch.float32) if q else None
    d = lib.rmsnorm_desc(rows, c, mx.ptr, mo.ptr, lib.DT_E4M3 if q else lib.DT_F16, eps, mr.ptr if mr else None,
                         mw.ptr if mw else None, ms.ptr if ms else None, msc.ptr if q else None,
                         strides[0], strides[1], strides[2], strides[3])
    torch.cuda.synchronize()
    lib.rmsnorm(d, stream)
    torch.cuda.synchronize()
    return mo.check(), msc.check()[0] if q else None, ms.check() if ms else None


SIZES = [(1, 1), (3, 2), (5, 9), (1000, 32), (77, 96), (129, 255), (33, 256), (19, 264), (7, 513), (9, 1000), (6, 1024),
         (3, 1025), (2, 4096), (1, 4096), (150, 2056), (4, 5001), (160, 5001), (2, 8191), (2, 16384), (149, 8200), (1, 32768),
         (2, 33001), (1, 70001), (150, 40000), (1000, 29), (3000, 3), (4100, 1), (2049, 2), (700, 130), (65, 254), (16, 255),
         (17, 255), (5000, 7)]


@pytest.mark.parametrize("q", [False, True], ids=["f16", "e4m3"])
@pytest.mark.parametrize("rows,c", SIZES)
def test_sizes(rows, c, q):
    x, r, w = normal(1, rows, c), normal(2, rows, c, scale=2.0), 1.0 + normal(3, c, dtype=torch.float32, scale=0.2)
    w = w.half()
    out, scale, s = run(x, r, w, q, keep_sum=True)
    h, y = reference(x, r, w)
    check_out(out, scale, y)
    # the sum of two binary16 values in 32 bits, rounded again: 2^-11 for the last rounding, 2^-24 for the first
    assert_within(s, h, h.abs() * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25, "sum")


@pytest.mark.parametrize("q", [False, True], ids=["f16", "e4m3"])
@pytest.mark.parametrize("residual,weight,keep", [(False, False, False), (False, True, True), (True, False, False), (True, True, False)])
@pytest.mark.parametrize("rows,c", [(37, 64), (5, 777), (3, 4096)])
def test_optional_operands(rows, c, residual, weight, keep, q):
    x = normal(4, rows, c)
    r = normal(5, rows, c) if residual else None
    w = normal(6, c) if weight else None
    out, scale, s = run(x, r, w, q, keep_sum=keep)
    h, y = reference(x, r, w)
    check_out(out, scale, y)
    if keep:
        assert_within(s, h, h.abs() * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25, "sum")


@pytest.mark.parametrize("q", [False, True], ids=["f16", "e4m3"])
@pytest.mark.parametrize("strides,offsets", [((72, 80, 88, 96), (0, 8, 16, 0)), ((68, 68, 68, 68), (4, 0, 4, 4)),
                                             ((66, 70, 74, 66), (2, 2, 0, 2)), ((65, 67, 69, 71), (1, 0, 3, 5)),
                                             ((64, 64, 64, 1001), (0, 0, 0, 1))])
@pytest.mark.parametrize("wide", [1, 32, 700])
def test_strides_and_alignment(strides, offsets, q, wide):
    """Windows of wider rows, at offsets that leave 16, 8, 4 or 2 byte accesses, in each of the kernel's forms."""
    rows, c = 21 if wide < 700 else 3, 64 * wide
    strides = tuple(s - 64 + c for s in strides)
    x, r, w = normal(7, rows, c), normal(8, rows, c), normal(9, c)
    out, scale, s = run(x, r, w, q, keep_sum=True, strides=strides, offsets=offsets)
    h, y = reference(x, r, w)
    check_out(out, scale, y)
    assert_within(s, h, h.abs() * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25, "sum")


@pytest.mark.parametrize("rows,c", [(9, 48), (300, 27), (7, 1000), (3, 4096), (2, 5001), (2, 40001)])
def test_in_place(rows, c):
    """The sum over the residual and the output over x, as a block of layers keeps its buffers."""
    x, r, w = normal(10, rows, c), normal(11, rows, c), normal(12, c)
    mx, mr, mw = Mat(rows, c, data=x), Mat(rows, c, data=r), Mat(1, c, data=w[None])
    lib.rmsnorm(lib.rmsnorm_desc(rows, c, mx.ptr, mx.ptr, eps=EPS, residual=mr.ptr, weight=mw.ptr, sum_out=mr.ptr))
    torch.cuda.synchronize()
    h, y = reference(x, r, w)
    check_out(mx.check(), None, y)
    assert_within(mr.check(), h, h.abs() * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25, "sum")


@pytest.mark.parametrize("c", [24, 37, 640, 4096, 5001, 40001])
def test_rows_that_are_not_finite_or_zero(c):
    """NaN, infinity, zeros, the type's lowest value and its smallest, each in a row of its own; other rows untouched."""
    low = torch.finfo(torch.float16).min
    x = normal(13, 7, c)
    x[1, c // 2] = float("nan")
    x[2, c - 1] = float("inf")
    x[3] = 0.0
    x[4] = low
    x[5] = 2.0 ** -24
    w = normal(14, c) + 2.0
    h, y = reference(x, None, w)
    out, _, _ = run(x, None, w)
    # binary16: what the formula gives: NaN everywhere in the NaN row; inf * 0 at the infinity and 0 beside it
    assert_within(out, y, tol_f16(y), "out")
    out, scale, _ = run(x, None, w, q=True)
    fine = [0, 3, 4, 5, 6]
    check_out(out[fine], scale[fine], y[fine])
    assert scale[3] == 1.0 and not out[3].any()
    assert torch.isnan(out[1:3]).all() and torch.isnan(scale[1:3]).all()
    # all lowest values, twice: the 32 bit sum is fine, its binary16 rounding is minus infinity
    lowest = torch.full((1, c), low, dtype=torch.float16)
    out, _, s = run(lowest, lowest, None, keep_sum=True)
    assert torch.isinf(s).all() and (s < 0).all()
    check_out(out, None, torch.full((1, c), -1.0, dtype=torch.float64))


@pytest.mark.parametrize("c", [16, 4096])
def test_eps(c):
    x = normal(15, 4, c, scale=1e-3)
    for eps in (1e-12, 1e-5, 1.0):
        out, _, _ = run(x, eps=eps)
        check_out(out, None, reference(x, None, None, eps)[1])


def test_streams_and_graph():
    """Two calls at once on two streams, and a captured call replayed on new values: the same bits as alone."""
    rows, c = 64, 2048
    xs = [normal(20 + i, rows, c).cuda() for i in range(2)]
    alone, outs = [], []
    for x in xs:
        o = torch.empty_like(x)
        lib.rmsnorm(lib.rmsnorm_desc(rows, c, x.data_ptr(), o.data_ptr()))
        torch.cuda.synchronize()
        alone.append(o.clone())
    streams = [torch.cuda.Stream() for _ in xs]
    for x, st in zip(xs, streams):
        o = torch.empty_like(x)
        outs.append(o)
        st.wait_stream(torch.cuda.current_stream())
        for _ in range(20):
            lib.rmsnorm(lib.rmsnorm_desc(rows, c, x.data_ptr(), o.data_ptr()), st.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(alone, outs))
    x, o = torch.empty_like(xs[0]), torch.empty_like(xs[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lib.rmsnorm(lib.rmsnorm_desc(rows, c, x.data_ptr(), o.data_ptr()), torch.cuda.current_stream().cuda_stream)
    for src, want in zip(xs, alone):
        x.copy_(src)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want)


def test_offsets_past_32_bits():
    """The last row of a tensor of more than 2^32 elements (rows far apart in one buffer)."""
    rows, c, stride = 3, 72, 1 << 31
    buf = torch.zeros(2 * stride + c, dtype=torch.float16, device="cuda")
    x = normal(30, rows, c)
    view = torch.as_strided(buf, (rows, c), (stride, 1))
    view.copy_(x)
    out = torch.empty(rows, c, dtype=torch.float16, device="cuda")
    lib.rmsnorm(lib.rmsnorm_desc(rows, c, buf.data_ptr(), out.data_ptr(), x_stride=stride))
    torch.cuda.synchronize()
    check_out(out.cpu().double(), None, reference(x, None, None)[1])


def test_buffers_of_another_place_are_refused():
    x = torch.zeros(4, 8, dtype=torch.float16)
    y = torch.zeros(4, 8, dtype=torch.float16, device="cuda")
    for a, b in ((x, y), (y, x)):
        d = lib.rmsnorm_desc(4, 8, a.data_ptr(), b.data_ptr())
        assert lib.L.dnxcu_rmsnorm_launch(d, None) == lib.E_BAD_ARG
    torch.cuda.synchronize()
