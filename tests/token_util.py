"""Helpers for the tests of the linear layer and the root-mean-square norm: matrices laid out in guarded buffers."""
import torch

CANARY = {torch.float16: 12345.0, torch.float32: 1.2345e30, torch.float8_e4m3fn: 208.0}


class Mat:
    """rows x cols elements at `stride` elements per row, `offset` elements into a buffer that is filled with a canary:
    whatever a kernel writes outside the rows shows up in check()."""

    def __init__(self, rows, cols, dtype=torch.float16, stride=None, offset=0, data=None):
        self.rows, self.cols, self.stride = rows, cols, stride or cols
        pad = 1024
        n = (rows - 1) * self.stride + cols
        self.buf = torch.full((n + 2 * pad + offset,), CANARY[dtype], dtype=torch.float32).to(dtype).cuda()
        self.view = torch.as_strided(self.buf, (rows, cols), (self.stride, 1), pad + offset)
        if data is not None:
            self.view.copy_(data.to(dtype))
        elif dtype != torch.float8_e4m3fn:
            self.view.fill_(float("nan"))  # what stays unwritten is caught by the comparison
        self.before = self.buf.clone()

    @property
    def ptr(self):
        return self.view.data_ptr()

    def check(self):
        """Nothing outside the rows has changed; returns the rows on the host, in 64 bits."""
        bits = {2: torch.int16, 4: torch.int32, 1: torch.uint8}[self.buf.element_size()]
        now, before = self.buf.view(bits).cpu().clone(), self.before.view(bits).cpu().clone()
        off = self.view.storage_offset()
        for t in (now, before):
            torch.as_strided(t, (self.rows, self.cols), (self.stride, 1), off).zero_()
        assert torch.equal(now, before), "written outside the rows"
        return self.view.to(torch.float32).cpu().double()


def normal(seed, *shape, dtype=torch.float16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def assert_within(got, ref, tol, what=""):
    """|got - ref| <= tol element by element; NaN and infinities in the same places."""
    assert got.shape == ref.shape, what
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN in other places"
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]), f"{what}: infinities differ"
    d = (got - ref).abs()[fin]
    t = tol[fin]
    bad = ~(d <= t)
    if bad.any():
        i = torch.argmax(torch.where(bad, d / t, torch.zeros_like(d)))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst |d|={d[i]:.3g} tol={t[i]:.3g} "
                             f"ref={ref[fin][i]:.6g}")
