"""The operators together, as a residual block runs them: norm with the residual's addition to 8 bits, a widening layer on
the 8 bit rows, a narrowing layer that adds the residual stream back, and the next block's norm on it — one stream, one
graph.  Every stage is held against its formula in 64 bits on what the stage before it gave."""
import math

import pytest
import torch

from denox_b200 import lib
from test_linear_gpu import reference
from test_rmsnorm_gpu import EPS, check_out, reference as norm_reference
from token_util import assert_within, normal

pytestmark = pytest.mark.gpu


def e4m3_weights(seed, n, k):
    w = normal(seed, n, k, dtype=torch.float32, scale=1 / math.sqrt(k))
    s = w.abs().amax(1) / 448.0
    return (w / s[:, None]).to(torch.float8_e4m3fn).cuda(), s.cuda()


@pytest.mark.parametrize("rows,c,wide", [(1, 256, 1024), (9, 512, 1536), (77, 384, 1000), (600, 1024, 4096), (1088 * 24, 64, 96), (130, 33, 65)])
def test_block(rows, c, wide):
    half = dict(dtype=torch.float16, device="cuda")
    x, stream = normal(1, rows, c).cuda(), normal(2, rows, c).cuda()
    g1, g2 = (1.0 + normal(3, c, dtype=torch.float32, scale=0.2)).half().cuda(), normal(4, c).cuda()
    w1, s1 = e4m3_weights(5, wide, c)
    w2, b1, b2 = normal(6, c, wide, scale=1 / math.sqrt(wide)).cuda(), normal(7, wide).cuda(), normal(8, c).cuda()
    residual = torch.empty(rows, c, **half)
    q, qs = torch.empty(rows, c, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(rows, dtype=torch.float32, device="cuda")
    mid, out = torch.empty(rows, wide, **half), torch.empty(rows, c, **half)
    p = lambda t: t.data_ptr()
    norm1 = lib.rmsnorm_desc(rows, c, p(x), p(q), lib.DT_E4M3, EPS, p(residual), p(g1), p(residual), p(qs))
    up = lib.LinearPlan(lib.linear_desc(rows, c, wide, p(q), p(w1), p(mid), lib.DT_E4M3, lib.ACT_SILU, x_scale=p(qs), w_scale=p(s1), bias=p(b1)))
    down = lib.LinearPlan(lib.linear_desc(rows, wide, c, p(mid), p(w2), p(residual), bias=p(b2), residual=p(residual)))
    norm2 = lib.rmsnorm_desc(rows, c, p(residual), p(out), eps=EPS, weight=p(g2))

    def block(st):
        lib.rmsnorm(norm1, st)
        up.launch(st)
        down.launch(st)
        lib.rmsnorm(norm2, st)

    # stage by stage
    residual.copy_(stream)
    lib.rmsnorm(norm1)
    torch.cuda.synchronize()
    h, y = norm_reference(x.cpu(), stream.cpu(), g1.cpu())
    check_out(q.float().cpu().double(), qs.cpu().double(), y)
    after_add = residual.clone()
    up.launch()
    torch.cuda.synchronize()
    ref, tol = reference(q, w1, qs, s1, b1, act="silu")
    assert_within(mid.cpu().double(), ref, tol, "up")
    down.launch()
    torch.cuda.synchronize()
    ref, tol = reference(mid, w2, bias=b2, residual=after_add)
    assert_within(residual.cpu().double(), ref, tol, "down")
    lib.rmsnorm(norm2)
    torch.cuda.synchronize()
    check_out(out.cpu().double(), None, norm_reference(residual.cpu(), None, g2.cpu())[1])
    want = out.clone(), residual.clone()
    # at once, and replayed: the same bits
    for _ in range(3):
        residual.copy_(stream)
        block(0)
    torch.cuda.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(residual, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        residual.copy_(stream)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(residual, want[1])
    del graph
    up.close()
    down.close()


def test_every_kernel_at_once_on_three_streams():
    """Chains of all the kernels (row, split, single and paired tiles, unaligned plans, norms) on three streams at once: the
    bits of each alone."""
    half = dict(dtype=torch.float16, device="cuda")
    p = lambda t: t.data_ptr()
    shapes = [(1, 512, 700), (40, 4096, 512), (200, 256, 1024), (2560, 512, 3840), (300, 257, 129), (5000, 32, 48)]
    keep, chains = [], []
    for k in range(3):
        chain = []
        for i, (m, c, n) in enumerate(shapes[k:] + shapes[:k]):
            x, w, b = normal(10 * i + k, m, c).cuda(), normal(10 * i + k + 5, n, c, scale=1 / math.sqrt(c)).cuda(), normal(i, n).cuda()
            mid, out, scale = torch.empty(m, n, **half), torch.empty(m, n, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(m, device="cuda")
            plan = lib.LinearPlan(lib.linear_desc(m, c, n, p(x), p(w), p(mid), bias=p(b), activation=lib.ACT_GELU))
            norm = lib.rmsnorm_desc(m, n, p(mid), p(out), lib.DT_E4M3, EPS, out_scale=p(scale))
            keep += [x, w, b]
            chain.append((plan, norm, mid, out, scale))
        chains.append(chain)

    def launch(chain, st):
        for plan, norm, *_ in chain:
            plan.launch(st)
            lib.rmsnorm(norm, st)

    bits = lambda chain: [t.view(torch.uint8).clone() for c in chain for t in c[2:]]
    torch.cuda.synchronize()
    want = []
    for chain in chains:
        launch(chain, 0)
        torch.cuda.synchronize()
        want.append(bits(chain))
    streams = [torch.cuda.Stream() for _ in chains]
    for _ in range(15):
        for chain, st in zip(chains, streams):
            launch(chain, st.cuda_stream)
    torch.cuda.synchronize()
    for chain, w in zip(chains, want):
        assert all(torch.equal(a, b) for a, b in zip(bits(chain), w))
    for chain in chains:
        for plan, *_ in chain:
            plan.close()


def test_capture_with_a_fork_and_a_join():
    """Two layers on forked streams between two others, captured into one graph: every edge holds."""
    half = dict(dtype=torch.float16, device="cuda")
    p = lambda t: t.data_ptr()
    m, c = 700, 512
    x, w = normal(1, m, c).cuda(), [normal(2 + i, c, c, scale=1 / math.sqrt(c)).cuda() for i in range(4)]
    a, b1, b2, out = (torch.empty(m, c, **half) for _ in range(4))
    layer = lambda src, i, dst, res=None: lib.LinearPlan(lib.linear_desc(m, c, c, p(src), p(w[i]), p(dst), residual=p(res) if res is not None else None))
    plans = [layer(x, 0, a), layer(a, 1, b1), layer(a, 2, b2), layer(b1, 3, out, b2)]
    for q in plans:
        q.launch()
        torch.cuda.synchronize()
    want = [t.clone() for t in (a, b1, b2, out)]
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        main = torch.cuda.current_stream()
        plans[0].launch(main.cuda_stream)
        side.wait_stream(main)
        plans[1].launch(main.cuda_stream)
        plans[2].launch(side.cuda_stream)
        main.wait_stream(side)
        plans[3].launch(main.cuda_stream)
    for _ in range(10):
        for t in (a, b1, b2, out):
            t.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t, v) for t, v in zip((a, b1, b2, out), want))
    # and without a graph
    for _ in range(10):
        for t in (a, b1, b2, out):
            t.fill_(float("nan"))
        main = torch.cuda.current_stream()
        plans[0].launch(main.cuda_stream)
        side.wait_stream(main)
        plans[1].launch(main.cuda_stream)
        plans[2].launch(side.cuda_stream)
        main.wait_stream(side)
        plans[3].launch(main.cuda_stream)
        torch.cuda.synchronize()
        assert all(torch.equal(t, v) for t, v in zip((a, b1, b2, out), want))
    del g
    for q in plans:
        q.close()
