"""Linear layer on the GPU against its formula in 64 bits.

Tolerances.  The products of two binary16 or e4m3 values are exact in 32 bits; a sum of K of them, added in 32 bits in any
order and with any rounding (the tensor cores may cut where others round: one unit, 2^-23), is off by at most
(K + 32) 2^-23 sum|x w|.  An activation's slope is below 1.2, so that error grows by 1.2 at most; the activation itself is
off by a few units plus, through the fast exponential, about two units per unit of its argument: |a| (16 + 2 |z|) 2^-23,
and 4 |z| 2^-24 for the 1 + erf of a negative argument.  The residual's addition is one 32 bit rounding, the output's
rounding half a step of binary16: 2^-11 |out| (2^-25 below its normal range).
Sums of small whole numbers are exact in every order: those tests ask for equal bits."""
import ctypes as C
import math

import pytest
import torch

from denox_b200 import lib
from token_util import Mat, assert_within, normal

pytestmark = pytest.mark.gpu

ACTS = {"none": lib.ACT_NONE, "relu": lib.ACT_RELU, "leaky": lib.ACT_LEAKY, "gelu": lib.ACT_GELU,
        "gelu_tanh": lib.ACT_GELU_TANH, "silu": lib.ACT_SILU}
VARIANTS = {"auto": lib.LINEAR_AUTO, "rows": lib.LINEAR_ROWS, "split": lib.LINEAR_SPLIT, "tile": lib.LINEAR_TILE,
            "any": lib.LINEAR_ANY}
ALPHA = 0.125


def activation(z, act):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "leaky":
        return torch.where(z > 0, z, ALPHA * z)
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(-z * math.sqrt(0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def reference(x, w, xs=None, ws=None, bias=None, residual=None, act="none"):
    """(result, tolerance) in 64 bits."""
    xd, wd = x.double().cuda(), w.double().cuda()
    s, a = xd @ wd.t(), xd.abs() @ wd.abs().t()
    scale = torch.ones(1, 1, dtype=torch.float64, device="cuda")
    if xs is not None:
        scale = scale * xs.double().cuda()[:, None]
    if ws is not None:
        scale = scale * ws.double().cuda()[None, :]
    z, mag = s * scale, a * scale.abs()
    if bias is not None:
        z = z + bias.double().cuda()
    y = activation(z, act)
    out = y if residual is None else y + residual.double().cuda()
    k = x.shape[1]
    tol = 1.2 * (k + 32) * 2.0 ** -23 * (mag + (z - s * scale).abs()) + y.abs() * (16 + 2 * z.abs()) * 2.0 ** -23 \
        + z.abs() * 2.0 ** -22 + (out.abs() + y.abs()) * 2.0 ** -24 + out.abs() * (2.0 ** -11 + 2.0 ** -20) + 2.0 ** -25
    # An infinite sum has no error, and an activation that is finite there is so exactly (relu of minus infinity is 0): what
    # is left is the residual's addition to that value and the output's rounding.
    tol = torch.where(torch.isinf(z) & torch.isfinite(out), out.abs() * (2.0 ** -11 + 2.0 ** -20) + 2.0 ** -25, tol)
    return out.cpu(), tol.cpu()


def run(x, w, xs=None, ws=None, bias=None, residual=None, act="none", variant="auto", strides=(0, 0, 0, 0),
        offsets=(0, 0, 0, 0), in_place=False, planned=False, stream=0, status=None):
    m, k = x.shape
    n = w.shape[0]
    f8 = x.dtype == torch.float8_e4m3fn
    pick = lambda i: dict(stride=strides[i] or None, offset=offsets[i])
    mx, mw = Mat(m, k, x.dtype, data=x, **pick(0)), Mat(n, k, w.dtype, data=w, **pick(1))
    mr = Mat(m, n, data=residual, **pick(2)) if residual is not None else None
    mo = mr if in_place else Mat(m, n, **pick(3))
    vec = lambda v, dt: Mat(1, v.numel(), dt, data=v[None]) if v is not None else None
    mb, mxs, mws = vec(bias, torch.float16), vec(xs, torch.float32), vec(ws, torch.float32)
    p = lambda t: t.ptr if t is not None else None
    d = lib.linear_desc(m, k, n, mx.ptr, mw.ptr, mo.ptr, lib.DT_E4M3 if f8 else lib.DT_F16, ACTS[act], ALPHA, p(mxs),
                        p(mws), p(mb), p(mr), strides[0], strides[1], strides[2], strides[2] if in_place else strides[3],
                        VARIANTS[variant], status)
    torch.cuda.synchronize()
    if planned:
        plan = lib.LinearPlan(d)
        plan.launch(stream)
        plan.launch(stream)
        torch.cuda.synchronize()
        plan.close()
    else:
        lib.linear(d, stream)
    torch.cuda.synchronize()
    for t in (mx, mw, mr if not in_place else None):
        if t is not None:
            t.check()
    return mo.check()


def e4m3(seed, rows, k):
    t = normal(seed, rows, k, dtype=torch.float32)
    s = t.abs().amax(1).clamp_min(1e-6) / 448.0
    return (t / s[:, None]).to(torch.float8_e4m3fn), s


def operands(dtype, m, k, n, seed=1):
    if dtype == "f16":
        return normal(seed, m, k), normal(seed + 1, n, k, scale=1 / math.sqrt(k)), None, None
    x, xs = e4m3(seed, m, k)
    w, ws = e4m3(seed + 1, n, k)
    return x, w, xs, ws / math.sqrt(k)


# (variant, rows, c_in, c_out): every variant on, one below and one above its tile borders
SIZES = [("rows", 1, 16, 1), ("rows", 1, 64, 16), ("rows", 2, 4096, 33), ("rows", 8, 1040, 100), ("rows", 9, 2064, 48),
         ("rows", 16, 4096, 130),
         ("split", 1, 16, 8), ("split", 1, 4096, 256), ("split", 16, 128, 128), ("split", 17, 160, 129), ("split", 100, 2048, 1000),
         ("split", 128, 272, 127), ("split", 250, 1024, 256), ("split", 257, 64, 300), ("split", 600, 528, 96),
         ("tile", 1, 16, 8), ("tile", 127, 64, 64), ("tile", 128, 128, 128), ("tile", 129, 144, 136), ("tile", 300, 80, 16),
         ("tile", 1000, 208, 96), ("tile", 513, 1024, 999), ("tile", 700, 32, 40), ("tile", 1000, 64, 33), ("tile", 1, 16, 63), ("tile", 333, 48, 1), ("tile", 20000, 64, 50), ("tile", 2048, 512, 4736), ("tile", 5000, 256, 2305),
         ("any", 1, 1, 1), ("any", 3, 9, 5), ("any", 1000, 9, 32), ("any", 129, 65, 127), ("any", 257, 1001, 129), ("any", 130, 130, 300),
         ("auto", 1, 4096, 4096), ("auto", 12, 3000, 777), ("auto", 64, 77, 77), ("auto", 5, 8, 3), ("auto", 4099, 1024, 1024)]


@pytest.mark.parametrize("dtype", ["f16", "e4m3"])
@pytest.mark.parametrize("variant,m,k,n", SIZES)
def test_sizes_whole_numbers(variant, m, k, n, dtype):
    """Whole numbers whose sums every order of addition gives exactly: the bits have to be right."""
    g = torch.Generator().manual_seed(m * 7 + k)
    t = torch.float16 if dtype == "f16" else torch.float8_e4m3fn
    x = torch.randint(-2, 3, (m, k), generator=g).float()
    w = torch.randint(-1, 2, (n, k), generator=g).float()
    # (a few ones per weight row only, so that sums stay below 2048, where binary16 holds every whole number)
    keep = torch.rand(n, k, generator=g) < min(1.0, 600.0 / k)
    w = w * keep
    bias = torch.randint(-8, 9, (n,), generator=g).half()
    residual = torch.randint(-100, 101, (m, n), generator=g).half()
    ref = x.double() @ w.double().t() + bias.double() + residual.double()
    assert float(ref.abs().max()) <= 2048
    got = run(x.to(t), w.to(t), bias=bias, residual=residual, variant=variant)
    assert torch.equal(got, ref)


@pytest.mark.parametrize("dtype", ["f16", "e4m3"])
@pytest.mark.parametrize("variant,m,k,n", SIZES)
def test_sizes(variant, m, k, n, dtype):
    x, w, xs, ws = operands(dtype, m, k, n)
    bias = normal(3, n)
    got = run(x, w, xs, ws, bias, act="silu" if n % 2 else "none", variant=variant)
    ref, tol = reference(x, w, xs, ws, bias, act="silu" if n % 2 else "none")
    assert_within(got, ref, tol)


@pytest.mark.parametrize("variant,m,k,n", [("rows", 3, 64, 40), ("split", 20, 64, 136), ("tile", 200, 64, 136), ("any", 70, 33, 71)])
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("residual", [False, True])
def test_epilogues(variant, m, k, n, act, residual):
    x, w, _, _ = operands("f16", m, k, n, 11)
    x = x * 4
    bias, r = normal(13, n), normal(14, m, n) if residual else None
    xs, ws = 0.5 + torch.rand(m, generator=torch.Generator().manual_seed(5)), 0.5 + torch.rand(n, generator=torch.Generator().manual_seed(6))
    for kw in (dict(), dict(bias=bias), dict(xs=xs), dict(ws=ws, bias=bias)):
        got = run(x, w, residual=r, act=act, variant=variant, **kw)
        ref, tol = reference(x, w, residual=r, act=act, **kw)
        assert_within(got, ref, tol, str(list(kw)))


@pytest.mark.parametrize("dtype", ["f16", "e4m3"])
@pytest.mark.parametrize("variant", ["rows", "split", "tile", "any"])
def test_strides(variant, dtype):
    """Windows of wider rows: on 16 byte boundaries for the copy engine, and at odd places for the output and residual."""
    m, k, n = 13, 96, 70
    x, w, xs, ws = operands(dtype, m, k, n, 21)
    r, b = normal(23, m, n), normal(24, n)
    ref, tol = reference(x, w, xs, ws, b, r, "gelu")
    for strides, offsets in (((112, 128, 72, 80), (16, 32, 8, 16)), ((96, 96, 71, 73), (0, 0, 1, 3)), ((160, 96, 80, 71), (0, 16, 0, 0)),
                             ((96, 96, 75, 72), (0, 0, 0, 0))):
        assert_within(run(x, w, xs, ws, b, r, "gelu", variant, strides, offsets), ref, tol, f"{strides} {offsets}")
    if variant == "any":
        for strides, offsets in (((97, 101, 70, 70), (1, 3, 0, 0)), ((98, 97, 71, 70), (2, 0, 0, 1))):
            assert_within(run(x, w, xs, ws, b, r, "gelu", variant, strides, offsets), ref, tol, f"{strides} {offsets}")
            assert_within(run(x, w, xs, ws, b, r, "gelu", "auto", strides, offsets), ref, tol, f"{strides} {offsets}")


@pytest.mark.parametrize("variant,m,k,n", [("rows", 4, 128, 72), ("split", 100, 128, 200), ("tile", 400, 128, 200), ("tile", 300, 64, 99),
                                           ("tile", 1001, 64, 37), ("any", 100, 77, 99), ("any", 300, 33, 33)])
def test_residual_in_place(variant, m, k, n):
    x, w, _, _ = operands("f16", m, k, n, 31)
    r = normal(33, m, n)
    ref, tol = reference(x, w, residual=r, act="relu")
    assert_within(run(x, w, residual=r, act="relu", variant=variant, in_place=True), ref, tol)


@pytest.mark.parametrize("variant,m,k,n", [("rows", 5, 128, 40), ("split", 40, 128, 140), ("tile", 150, 128, 140), ("any", 60, 65, 70)])
def test_values_that_are_not_finite(variant, m, k, n):
    """A NaN or an infinity in x reaches its row alone, one in the weights its column alone; what lies between the rows of
    a strided operand (NaN here) reaches nothing."""
    x, w, _, _ = operands("f16", m, k, n, 41)
    x[1, 3] = float("nan")
    x[2, k - 1] = float("inf")
    w[:, k - 1] = w[:, k - 1].abs() + 0.5
    w[4, 0] = float("nan")
    for act in ("none", "relu", "leaky"):
        ref, tol = reference(x, w, act=act)
        assert_within(run(x, w, act=act, variant=variant), ref, tol, act)
    big = torch.full_like(x, 60000.0)
    ones = torch.ones_like(w)
    assert torch.isinf(run(big, ones, variant=variant)).all()  # sums beyond binary16
    low = torch.full((m, n), torch.finfo(torch.float16).min, dtype=torch.float16)
    got = run(torch.zeros_like(x), torch.zeros_like(w), residual=low, variant=variant)
    assert torch.equal(got, low.double())


@pytest.mark.parametrize("variant,k", [("split", 72), ("split", 70), ("split", 65), ("tile", 72), ("tile", 70), ("tile", 65), ("rows", 80),
                                       ("any", 65), ("auto", 65), ("auto", 70)])
def test_garbage_between_rows(variant, k):
    """Channels beyond c_in (the rest of a padded row) are never multiplied, whatever they hold."""
    m, n = 9, 33
    x, w, _, _ = operands("f16", m, k, n, 51)
    wide = torch.full((m, 160), float("nan"), dtype=torch.float16, device="cuda")
    ww = torch.full((n, 160), float("inf"), dtype=torch.float16, device="cuda")
    wide[:, :k], ww[:, :k] = x.cuda(), w.cuda()
    out = torch.empty(m, n, dtype=torch.float16, device="cuda")
    lib.linear(lib.linear_desc(m, k, n, wide.data_ptr(), ww.data_ptr(), out.data_ptr(), x_stride=160, w_stride=160,
                               variant=VARIANTS[variant]))
    torch.cuda.synchronize()
    ref, tol = reference(x, w)
    assert_within(out.cpu().double(), ref, tol)


def test_plan_streams_and_graph():
    """A plan launched twice, on two streams at once and from a replayed graph gives the bits of one direct call."""
    for m, k, n in ((1, 512, 300), (40, 1024, 300), (600, 256, 1100)):
        x, w, _, _ = operands("f16", m, k, n, 61)
        want = run(x, w)
        assert torch.equal(run(x, w, planned=True), want)
        xd, wd = x.cuda(), w.cuda()
        outs = [torch.empty(m, n, dtype=torch.float16, device="cuda") for _ in range(3)]
        plans = [lib.LinearPlan(lib.linear_desc(m, k, n, xd.data_ptr(), wd.data_ptr(), o.data_ptr())) for o in outs]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for _ in range(10):
            for p, st in zip(plans, streams):
                p.launch(st.cuda_stream)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            plans[2].launch(torch.cuda.current_stream().cuda_stream)
        for _ in range(2):
            outs[2].zero_()
            g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o.cpu().double(), want)


@pytest.mark.parametrize("dtype", ["f16", "e4m3"])
@pytest.mark.parametrize("m,k,n,strides,offsets", [(17, 9, 5, (0, 0), (0, 0)), (130, 65, 300, (0, 0), (0, 0)), (100, 1001, 129, (0, 0), (0, 0)),
                                                   (1000, 27, 24, (0, 0), (0, 0)), (300, 64, 96, (65, 64), (0, 0)),
                                                   (300, 64, 96, (64, 67), (0, 0)), (257, 96, 64, (96, 96), (3, 0)),
                                                   (600, 513, 2000, (520, 515), (1, 5)), (1, 77, 40, (0, 0), (1, 1)),
                                                   (9, 333, 20, (0, 0), (0, 3)), (4000, 1, 1, (0, 0), (0, 0))])
def test_plan_of_unaligned_operands(m, k, n, strides, offsets, dtype):
    """What a kept plan does with rows off 16 byte boundaries (scratch), and a direct call without any: both right."""
    x, w, xs, ws = operands(dtype, m, k, n, 65)
    b, r = normal(66, n), normal(67, m, n)
    ref, tol = reference(x, w, xs, ws, b, r, "silu")
    for planned in (True, False):
        got = run(x, w, xs, ws, b, r, "silu", strides=strides + (0, 0), offsets=offsets + (0, 0), planned=planned)
        assert_within(got, ref, tol, f"planned={planned}")


# (rows, c_in, c_out, dtype) that AUTO takes several rows at a time: 8, 8 with rows left over, 2, 4, 8 bit operands
GROUPED = [(151552, 9, 32, "f16"), (151560 + 5, 9, 32, "f16"), (160003, 3, 16, "f16"), (152001, 3, 9, "f16"), (39999, 8, 8, "f16"),
           (76003, 12, 20, "f16"), (155555, 16, 16, "f16"), (151557, 27, 5, "f16"), (151999, 2, 8, "e4m3"), (160000, 30, 9, "e4m3")]


@pytest.mark.parametrize("m,k,n,dtype", GROUPED)
def test_thin_layers_over_many_rows(m, k, n, dtype):
    t = torch.float16 if dtype == "f16" else torch.float8_e4m3fn
    g = torch.Generator().manual_seed(m)
    x, w = torch.randint(-2, 3, (m, k), generator=g).to(t), torch.randint(-2, 3, (n, k), generator=g).to(t)
    bias, r = torch.randint(-8, 9, (n,), generator=g).half(), torch.randint(-100, 101, (m, n), generator=g).half()
    want = x.double() @ w.double().t() + bias.double() + r.double()
    for in_place in (False, True):
        assert torch.equal(run(x, w, bias=bias, residual=r, in_place=in_place), want)
    assert torch.equal(run(x, w, bias=bias, planned=True), want - r.double())
    ws = 0.5 + torch.rand(n, generator=g)
    x = normal(m, m, k, dtype=torch.float32).to(t)
    ref, tol = reference(x, w, ws=ws, bias=bias, act="gelu")
    assert_within(run(x, w, ws=ws, bias=bias, act="gelu"), ref, tol)


@pytest.mark.parametrize("m,k,n,dtype", GROUPED)
def test_thin_layers_keep_values_that_are_not_finite_in_their_row(m, k, n, dtype):
    t = torch.float16 if dtype == "f16" else torch.float8_e4m3fn
    x, w = normal(1, m, k, dtype=torch.float32).to(t), normal(2, n, k, dtype=torch.float32)
    w[:, 0] = w[:, 0].abs() + 0.5
    w = w.to(t)
    bias, r = normal(3, n), normal(4, m, n)
    for i, v in ((0, "nan"), (13, "inf"), (14, "-inf"), (m // 2, "nan"), (m - 1, "inf")):
        x[i, 0] = float(v) if dtype == "f16" else float("nan")
    for act in ("none", "relu"):
        ref, tol = reference(x, w, bias=bias, residual=r, act=act)
        got = run(x, w, bias=bias, residual=r, act=act)
        assert_within(got, ref, tol, act)
        assert_within(run(x, w, bias=bias, residual=r, act=act, in_place=True), ref, tol, act)


def test_offsets_past_32_bits():
    """Rows of x and of the output that lie more than 2^32 elements from the first."""
    m, k, n, stride = 3, 64, 48, (1 << 31) + 8
    x, w, _, _ = operands("f16", m, k, n, 71)
    buf = torch.zeros(2 * stride + 64, dtype=torch.float16, device="cuda")
    torch.as_strided(buf, (m, k), (stride, 1)).copy_(x)
    wd, out = w.cuda(), torch.zeros(m, n, dtype=torch.float16, device="cuda")
    ref, tol = reference(x, w)
    for v in ("rows", "split", "tile", "any"):
        out.zero_()
        lib.linear(lib.linear_desc(m, k, n, buf.data_ptr(), wd.data_ptr(), out.data_ptr(), x_stride=stride, variant=VARIANTS[v]))
        torch.cuda.synchronize()
        assert_within(out.cpu().double(), ref, tol, v)
    xd = x.cuda()
    for v in ("rows", "split", "tile", "any"):
        buf.zero_()
        lib.linear(lib.linear_desc(m, k, n, xd.data_ptr(), wd.data_ptr(), buf.data_ptr(), out_stride=stride, variant=VARIANTS[v]))
        torch.cuda.synchronize()
        assert_within(torch.as_strided(buf, (m, n), (stride, 1)).cpu().double(), ref, tol, v)


def test_status_stays_clear():
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    x, w, _, _ = operands("f16", 300, 256, 300, 81)
    for v in ("split", "tile", "any"):
        run(x, w, variant=v, status=st.data_ptr())
    assert int(st) == 0


def test_buffers_of_another_place_are_refused():
    h = torch.zeros(64, 64, dtype=torch.float16)
    d = torch.zeros(64, 64, dtype=torch.float16, device="cuda")
    e = torch.zeros(64, 64, dtype=torch.float16, device="cuda")
    for a, b, c in ((h, d, e), (d, h, e), (d, e, h)):
        r = lib.linear_desc(64, 64, 64, a.data_ptr(), b.data_ptr(), c.data_ptr())
        assert lib.L.dnxcu_linear_launch(r, None) == lib.E_BAD_ARG
        p = C.c_void_p()
        assert lib.L.dnxcu_linear_plan_create(r, C.byref(p)) == lib.E_BAD_ARG
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["f16", "e4m3"])
@pytest.mark.parametrize("variant,m,k,n", [("rows", 8, 8192, 64), ("split", 30, 8192, 128), ("tile", 200, 8192, 128), ("any", 40, 8191, 64),
                                           ("tile", 2560, 1024, 3840)])
def test_sums_are_held_in_32_bits(variant, m, k, n, dtype):
    """The residual takes the rounded sum away: what is left shows the sum's last bits."""
    t = torch.float16 if dtype == "f16" else torch.float8_e4m3fn
    x, w = normal(91, m, k, dtype=torch.float32).to(torch.float8_e4m3fn), normal(92, n, k, dtype=torch.float32).to(torch.float8_e4m3fn)
    x, w = x.to(torch.float32).to(t), w.to(torch.float32).to(t)
    s, _ = reference(x, w)
    ref, tol = reference(x, w, residual=(-s).half())
    assert_within(run(x, w, residual=(-s).half(), variant=variant), ref, tol)


def test_direct_call_in_a_capture_and_plans_made_during_one():
    m, k, n = 40, 513, 200
    x, w, _, _ = operands("f16", m, k, n, 95)
    ref, tol = reference(x, w)
    xd, wd = x.cuda(), w.cuda()
    outs = [torch.zeros(m, n, dtype=torch.float16, device="cuda") for _ in range(2)]
    descs = [lib.linear_desc(m, k, n, xd.data_ptr(), wd.data_ptr(), o.data_ptr()) for o in outs]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        st = torch.cuda.current_stream().cuda_stream
        lib.linear(descs[0], st)
        plan = lib.LinearPlan(descs[1])  # (unaligned: allocates its scratch)
        plan.launch(st)
    g.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert_within(o.cpu().double(), ref, tol)
    del g
    plan.close()


@pytest.mark.parametrize("variant,m,k,n", [("split", 64, 2048, 512), ("tile", 300, 2048, 512), ("tile", 2560, 512, 3840), ("any", 100, 1001, 300)])
def test_gives_up_cleanly_when_the_wait_limit_is_tiny(variant, m, k, n):
    """With a limit of one microsecond ordinary waits run out: the launch returns, the status word may hold the wait's code,
    and the device and the library are in order afterwards."""
    x, w, _, _ = operands("f16", m, k, n, 97)
    ref, tol = reference(x, w)
    xd, wd = x.cuda(), w.cuda()
    out, status = torch.zeros(m, n, dtype=torch.float16, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    d = lib.linear_desc(m, k, n, xd.data_ptr(), wd.data_ptr(), out.data_ptr(), variant=VARIANTS[variant], device_status=status.data_ptr())
    lib.check(lib.L.dnxcu_set_wait_limit_us(1))
    try:
        codes = []
        for _ in range(3):
            lib.linear(d)
            torch.cuda.synchronize()
            codes.append(int(status))
            status.zero_()
    finally:
        lib.check(lib.L.dnxcu_set_wait_limit_us(0))
    assert all(c == 0 or 11 <= c <= 15 for c in codes), codes
    lib.linear(d)
    torch.cuda.synchronize()
    assert int(status) == 0
    assert_within(out.cpu().double(), ref, tol)
