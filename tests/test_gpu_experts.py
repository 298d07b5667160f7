"""le_mm_experts and its gradients against the formula in 64 bits: whole numbers, whose sums fp32 holds exactly, so that every result has
to be the exact one rounded once; and real numbers within the bound of fp32 sums."""
import functools

import pytest

import lastengine_amd as le
from tests.test_gpu_graphs import capture

pytestmark = pytest.mark.gpu

TYPES = [le.F32, le.F16, le.BF16]


def dtype(ty):
    import torch
    return {le.F32: torch.float32, le.F16: torch.float16, le.BF16: torch.bfloat16}[ty]


def half_step(ty):
    import torch
    return torch.finfo(dtype(ty)).eps / 2


def whole(gen, *shape):
    import torch
    return torch.randint(-4, 5, shape, generator=gen, dtype=torch.float64)


def real(gen, *shape):
    import torch
    return torch.randn(*shape, generator=gen, dtype=torch.float64)


class Rows:
    """(n, width) rows `stride` values apart from a point `at` values into a buffer of `fill`."""

    def __init__(self, ty, n, width, stride=None, at=0, fill=float("nan")):
        import torch
        self.stride = stride or width
        self.flat = torch.full((at + n * self.stride + 64,), fill, dtype=dtype(ty), device="cuda")
        self.rows = self.flat[at:at + n * self.stride].view(n, self.stride)[:, :width]
        self.ptr = self.flat.data_ptr() + at * self.flat.element_size()

    def untouched(self, live, fill):
        """Whether everything but the first `live` rows is still `fill`."""
        other = self.flat.clone()
        first = (self.ptr - self.flat.data_ptr()) // self.flat.element_size()
        other[first:first + self.rows.shape[0] * self.stride].view(-1, self.stride)[:live, :self.rows.shape[1]] = fill
        return bool((other == fill).all())


class Case:
    def __init__(self, ty, counts, rows, cols, seed, make=whole, behind=3, gap=0, at=0, dw_ty=None):
        import torch
        gen = torch.Generator().manual_seed(seed)
        self.ty, self.dw_ty, self.counts, self.m, self.k = ty, ty if dw_ty is None else dw_ty, counts, rows, cols
        self.e, self.live = len(counts), sum(counts)
        self.n = self.live + behind
        t = dtype(ty)
        x, dy = make(gen, self.live, cols).to(t), make(gen, self.live, rows).to(t)
        w = make(gen, self.e, rows, cols).to(t)
        w[[i for i, c in enumerate(counts) if c == 0]] = float("nan")  # an expert without rows is in no result
        self.off = torch.tensor([0] + counts).cumsum(0).to(torch.int32).cuda()
        self.x, self.dy = Rows(ty, self.n, cols, cols + gap, at), Rows(ty, self.n, rows, rows + gap, at)
        self.w = Rows(ty, self.e, rows * cols, None, at)
        self.x.rows[:self.live] = x.cuda()
        self.dy.rows[:self.live] = dy.cuda()
        self.w.rows.copy_(w.reshape(self.e, -1))
        self.y, self.dx = (Rows(ty, self.n, c, c + gap, at, 77.0) for c in (rows, cols))
        self.dw = Rows(self.dw_ty, self.e, rows * cols, None, at, 77.0)
        self.x64, self.dy64, self.w64 = x.double(), dy.double(), w.double()

    def parts(self):
        i = 0
        for e, c in enumerate(self.counts):
            yield e, slice(i, i + c)
            i += c

    def want(self, x, dy, w):
        """y, dx and dw of these rows and weights, in 64 bits."""
        import torch
        y, dx, dw = torch.zeros(self.live, self.m).double(), torch.zeros(self.live, self.k).double(), torch.zeros(self.e, self.m, self.k).double()
        for e, s in self.parts():
            if s.stop > s.start:
                y[s], dx[s], dw[e] = x[s] @ w[e].t(), dy[s] @ w[e], dy[s].t() @ x[s]
        return y, dx, dw

    def run(self, engine, stream=None, ws=None):
        shape = (self.e, self.n, self.m, self.k)
        kw = dict(ldx=self.x.stride, ldy=self.y.stride, stream=stream)
        engine.mm_experts(self.ty, self.w.ptr, self.off, self.x.ptr, self.y.ptr, *shape, **kw)
        engine.mm_experts_dx(self.ty, self.w.ptr, self.off, self.dy.ptr, self.dx.ptr, *shape, **kw)
        engine.mm_experts_dw(self.ty, self.dy.ptr, self.x.ptr, self.off, self.dw.ptr, *shape, dw_ty=self.dw_ty, ws=ws, **kw)

    def got(self):
        import torch
        torch.cuda.synchronize()
        assert self.y.untouched(self.live, 77.0) and self.dx.untouched(self.live, 77.0) and self.dw.untouched(self.e, 77.0)
        return self.y.rows[:self.live].cpu(), self.dx.rows[:self.live].cpu(), self.dw.rows.cpu().reshape(self.e, self.m, self.k)

    def check_whole(self):
        import torch
        for name, got, want in zip(("y", "dx", "dw"), self.got(), self.want(self.x64, self.dy64, self.w64)):
            assert torch.equal(got, want.to(got.dtype)), name

    def check_real(self):
        """fp32 sums of n terms in any order, each step off by at most a last place (2^-23): n 2^-23 of the terms' magnitudes; then one
        rounding to the result's type (fp16's below its least normal: half of 2^-24)."""
        wants, mags = self.want(self.x64, self.dy64, self.w64), self.want(self.x64.abs(), self.dy64.abs(), self.w64.abs())
        for name, got, want, mag, n, ty in zip(("y", "dx", "dw"), self.got(), wants, mags, (self.k, self.m, max(self.counts)), (self.ty, self.ty, self.dw_ty)):
            bound = (n + 1) * 2.0 ** -23 * mag
            bound = bound + half_step(ty) * (want.abs() + bound) + (2.0 ** -25 if ty == le.F16 else 1e-38)
            assert ((got.double() - want).abs() <= bound).all(), name


SHAPES = [([1], 1, 1), ([1], 64, 64), ([0, 2, 0, 5, 0], 7, 5), ([3, 0, 1, 40], 33, 100), ([31, 33, 64], 128, 256), ([129, 0, 127, 1], 200, 136), ([300], 130, 72), ([20, 260], 515, 1001),
          ([0, 0], 40, 24), ([5, 9, 7], 512, 1024), ([1] * 70, 48, 96), ([17] * 9, 264, 520), ([700], 256, 384), ([2500], 24, 40),
          ([1, 0, 3, 2, 0, 0, 1, 0], 264, 136), ([1, 1, 0, 0, 2], 1000, 520), ([130, 0, 5, 64, 33, 1, 0, 2], 1000, 4088), ([40, 300] * 8, 1016, 1000),
          ([3000, 0, 1], 130, 264), ([1, 0, 2000, 63], 33, 515), ([9000], 129, 130),
          ([1] * 70, 1000, 2056), ([2, 0, 1, 0] * 32, 2100, 72), ([6, 12, 31, 40] + [0] * 50, 200, 2056), ([3, 20, 0, 7] + [0] * 20, 40, 2056),
          ([5] * 63 + [160], 2056, 72), ([1, 9] * 31 + [140], 40, 2064), ([3, 0, 300, 77] * 3, 264, 1000), ([400, 410, 0, 500], 2049, 41), ([400, 410, 0, 500], 41, 2049), ([49] * 88, 2049, 41),
          ([49] * 87 + [80], 41, 2049)]


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("counts,rows,cols", SHAPES)
def test_whole_numbers(engine, ty, counts, rows, cols):
    c = Case(ty, counts, rows, cols, 1)
    c.run(engine)
    c.check_whole()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("gap,at", [(8, 0), (3, 0), (0, 1), (8, 8), (16, 3)])
@pytest.mark.parametrize("counts,rows,cols", [([4, 0, 50], 96, 160), ([140, 3], 136, 264), ([3, 9], 50, 77), ([6, 0, 20, 1] + [0] * 240, 72, 152)])
def test_strides_and_alignment(engine, ty, gap, at, counts, rows, cols):
    """Rows apart, NaN between and around them, addresses aligned to their type alone."""
    c = Case(ty, counts, rows, cols, 2, gap=gap, at=at, behind=200)
    c.run(engine)
    c.check_whole()


@pytest.mark.parametrize("ty", [le.F16, le.BF16])
@pytest.mark.parametrize("counts,rows,cols", [([0, 2, 6], 40, 72), ([64, 100], 256, 256), ([1500], 64, 48), ([130, 0, 70, 3], 1000, 4088), ([900, 2000], 20, 131)])
def test_weights_gradient_in_fp32(engine, ty, counts, rows, cols):
    c = Case(ty, counts, rows, cols, 3, dw_ty=le.F32)
    c.run(engine)
    c.check_whole()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("counts,rows,cols", [([1, 2, 0, 5], 128, 2048), ([37, 90], 300, 515), ([500, 12], 256, 768), ([1800], 96, 64)])
def test_real_numbers(engine, ty, counts, rows, cols):
    c = Case(ty, counts, rows, cols, 4, make=real)
    c.run(engine)
    c.check_real()


@pytest.mark.parametrize("ty", TYPES)
def test_rows_that_are_not_finite_stay_alone(engine, ty):
    """A NaN in one row: that row of y and dx, that expert's dw. Infinite weights: that expert's rows."""
    import torch
    c = Case(ty, [3, 40, 6], 64, 96, 5)
    c.x.rows[10, 7] = float("nan")
    c.dy.rows[11, 9] = float("inf")
    c.run(engine)
    y, dx, dw = c.got()
    wy, wdx, wdw = (v.to(dtype(ty)) for v in c.want(c.x64, c.dy64, c.w64))
    assert torch.isnan(y[10]).all() and torch.equal(y[:10], wy[:10]) and torch.equal(y[11:], wy[11:])
    assert not torch.isfinite(dx[11]).any() and torch.equal(dx[:11], wdx[:11]) and torch.equal(dx[12:], wdx[12:])
    assert torch.equal(dw[0], wdw[0]) and torch.equal(dw[2], wdw[2])
    assert torch.isnan(dw[1][:, 7]).all() and not torch.isfinite(dw[1][9]).any()
    keep = torch.ones(64, 96, dtype=torch.bool)
    keep[:, 7], keep[9] = False, False
    assert torch.equal(dw[1][keep], wdw[1][keep])


@pytest.mark.parametrize("ty", TYPES)
def test_offsets_outside_the_buffers(engine, ty):
    """Rows are read and written within n_row whatever off holds."""
    import torch
    c = Case(ty, [4, 10, 6], 40, 72, 6, behind=0)
    c.off.copy_(torch.tensor([-9, 4, 14, 2000], dtype=torch.int32))
    c.run(engine)
    c.check_whole()


def test_no_rows(engine):
    c = Case(le.F16, [0, 0, 0], 24, 40, 7, behind=0)
    c.run(engine)
    c.check_whole()
    c = Case(le.F16, [0, 0, 0], 24, 40, 7, behind=50)
    c.run(engine)
    c.check_whole()


def test_many_experts(engine):
    import random
    r = random.Random(1)
    c = Case(le.BF16, [r.choice([0, 0, 0, 1, 2, 5]) for _ in range(1024)], 40, 72, 8)
    c.run(engine)
    c.check_whole()


@pytest.mark.parametrize("ty", [le.BF16, le.F32])
def test_rows_beyond_32_bits(engine, ty):
    """Row strides that put the last rows more than 2^32 values away, and an expert whose weights begin there."""
    import torch
    gen = torch.Generator().manual_seed(9)
    rows, cols, n, ld = 40, 72, 6, (1 << 30) + 8
    t = dtype(ty)
    big = [torch.empty(5 * ld + cols, dtype=t, device="cuda").as_strided((n, cols), (ld, 1)) for _ in range(2)]
    e = (1 << 32) // (rows * cols) + 2
    w = torch.empty(1024, (1 << 32) // 1024 + rows * cols, dtype=t, device="cuda").reshape(-1)
    rows2, cols2 = 2048, w.numel() // 1024 // 2048
    x, dy, we = whole(gen, n, cols).to(t), whole(gen, n, rows).to(t), whole(gen, 1, rows, cols).to(t)
    big[0].copy_(x)
    off = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    y, dw = torch.empty(n, rows, dtype=t, device="cuda"), torch.empty(1, rows, cols, dtype=t, device="cuda")
    wd = we.cuda()
    engine.mm_experts(ty, wd, off, big[0], y, 1, n, rows, cols, ldx=ld)
    engine.mm_experts_dx(ty, wd, off, dy.cuda(), big[1], 1, n, rows, cols, ldx=ld)
    engine.mm_experts_dw(ty, dy.cuda(), big[0], off, dw, 1, n, rows, cols, ldx=ld)
    assert torch.equal(y.cpu(), (x.double() @ we[0].double().t()).to(t))
    assert torch.equal(big[1].cpu(), (dy.double() @ we[0].double()).to(t))
    assert torch.equal(dw[0].cpu(), (dy.double().t() @ x.double()).to(t))
    del big
    # the last of 1024 experts, of 2048 x cols2 values each
    x, wl = whole(gen, 3, cols2).to(t), whole(gen, rows2, cols2).to(t)
    w[1023 * rows2 * cols2:1024 * rows2 * cols2] = wl.reshape(-1).cuda()
    off = torch.zeros(1025, dtype=torch.int32, device="cuda")
    off[1024] = 3
    assert 1023 * rows2 * cols2 > 1 << 31 and e
    y = torch.empty(3, rows2, dtype=t, device="cuda")
    engine.mm_experts(ty, w, off, x.cuda(), y, 1024, 3, rows2, cols2)
    assert torch.equal(y.cpu(), (x.double() @ wl.double().t()).to(t))
    engine.mm_experts_dx(ty, w, off, y, x2 := torch.empty(3, cols2, dtype=t, device="cuda"), 1024, 3, rows2, cols2)
    want = y.cpu().double() @ wl.double()
    # these sums can pass 2^24: fp32's bound as in check_real
    mag = y.cpu().double().abs() @ wl.double().abs()
    assert ((x2.cpu().double() - want).abs() <= half_step(ty) * want.abs() + 2 * rows2 * 2.0 ** -23 * mag).all()


@pytest.mark.parametrize("ty", TYPES)
def test_gradients_are_the_differences(engine, ty):
    """Whole numbers again: moving one input value by d moves sum(dy y) by d times its gradient, exactly (an input that appears in a linear
    form)."""
    import torch
    c = Case(ty, [3, 0, 6], 9, 13, 10, behind=0)
    c.run(engine)
    y0, dx, dw = (v.double() for v in c.got())
    for place in ((0, 0), (4, 12), (8, 5)):
        c.x.rows[place] += 2
        c.run(engine)
        assert float(((c.got()[0].double() - y0) * c.dy64).sum()) == 2 * float(dx[place])
        c.x.rows[place] -= 2
    for e, r, k in ((0, 0, 0), (2, 8, 12), (2, 3, 4)):
        c.w.rows[e, r * 13 + k] += 1
        c.run(engine)
        assert float(((c.got()[0].double() - y0) * c.dy64).sum()) == float(dw[e, r, k])
        c.w.rows[e, r * 13 + k] -= 1
    assert (dw[1] == 0).all() and torch.isfinite(dw).all()


def test_same_bits_from_call_to_call(engine):
    import torch
    for counts, rows, cols in (([300, 5, 0, 90], 200, 264), ([1, 2, 0, 8] * 20, 1000, 2056), ([2000], 48, 56), ([130, 0, 70, 3], 1000, 4088)):
        c = Case(le.BF16, counts, rows, cols, 11, make=real)
        c.run(engine)
        first = c.got()
        for _ in range(3):
            c.run(engine)
            assert all(torch.equal(a, b) for a, b in zip(first, c.got()))


def test_on_given_streams_and_in_graphs(engine):
    """Two captured steps replayed on two streams at once, with new inputs and eager calls between; then an eager call on a stream."""
    import torch
    cs = [Case(le.BF16, [40, 0, 200, 3], 136, 264, 12), Case(le.F32, [1800], 24, 40, 13)]
    wss = [torch.empty(max(16, engine.mm_experts_dw_workspace_size(c.ty, c.e, c.n, c.m, c.k)), dtype=torch.uint8, device="cuda") for c in cs]
    graphs = [capture(functools.partial(lambda c, ws, s: c.run(engine, s, ws), c, ws)) for c, ws in zip(cs, wss)]
    streams = [torch.cuda.Stream() for _ in cs]
    for rep in range(4):
        for c in cs:
            gen = torch.Generator().manual_seed(20 + rep)
            c.x64, c.dy64 = whole(gen, c.live, c.k), whole(gen, c.live, c.m)
            c.x.rows[:c.live], c.dy.rows[:c.live] = c.x64.to(c.x.rows.dtype).cuda(), c.dy64.to(c.x.rows.dtype).cuda()
            for r in (c.y, c.dx, c.dw):
                r.flat.fill_(77.0)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for c in cs:
            c.check_whole()
        cs[0].run(engine)
        cs[0].check_whole()
    cs[1].dw.flat.fill_(77.0)
    torch.cuda.synchronize()
    cs[1].run(engine, streams[0])
    cs[1].check_whole()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("at", [1, 2, 3, 8])
@pytest.mark.parametrize("counts,rows,cols", [([130, 0, 70, 3], 1000, 4088), ([33, 200, 0, 9], 1024, 4096), ([20, 260, 1], 520, 1000), ([1500], 64, 48), ([7, 3], 24, 40)])
def test_weights_gradient_aligned_to_its_type_alone(engine, ty, fp32, at, counts, rows, cols):
    """Rows of whole 16-byte pieces, so that the kernels of such rows run, and a result that begins anywhere."""
    import torch
    c = Case(ty, counts, rows, cols, 14, dw_ty=le.F32 if fp32 else None)
    c.dw = Rows(c.dw_ty, c.e, rows * cols, None, at, 77.0)
    c.run(engine)
    torch.cuda.synchronize()
    assert c.dw.untouched(c.e, 77.0)
    want = c.want(c.x64, c.dy64, c.w64)[2]
    assert torch.equal(c.dw.rows.cpu().reshape(want.shape), want.to(c.dw.rows.dtype))


def far_experts(ty, rows, cols, n_row, live, seed):
    """Weights of 1024 experts of which only the last is filled and has rows; its first value lies past 2^32."""
    import torch
    gen, t = torch.Generator().manual_seed(seed), dtype(ty)
    assert 1023 * rows * cols > 1 << 32
    w = torch.empty(1024 * rows * cols, dtype=t, device="cuda")
    wl, x, dy = whole(gen, rows, cols), whole(gen, live, cols), whole(gen, live, rows)
    w[1023 * rows * cols:] = wl.reshape(-1).to(t).cuda()
    off = torch.zeros(1025, dtype=torch.int32, device="cuda")
    off[1024] = live
    full = [torch.full((n_row, width), float("nan"), dtype=t, device="cuda") for width in (cols, rows)]
    full[0][:live], full[1][:live] = x.to(t).cuda(), dy.to(t).cuda()
    return w, off, full[0], full[1], wl, x, dy


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("rows,cols,n_row,live", [(2048, 2064, 3, 3), (2048, 2064, 4000, 300), (128, 32816, 4000, 300), (2048, 2065, 4000, 70), (2048, 2065, 50000, 300)])
def test_weights_past_32_bits(engine, ty, rows, cols, n_row, live):
    """Every way that y and dx read weights: few rows an expert, whole rows in narrow and wide tiles, rows of any alignment in small and
    large tiles."""
    import torch
    t = dtype(ty)
    w, off, x, dy, w64, x64, dy64 = far_experts(ty, rows, cols, n_row, live, 15)
    y, dx = (torch.full((n_row, width), 77.0, dtype=t, device="cuda") for width in (rows, cols))
    engine.mm_experts(ty, w, off, x, y, 1024, n_row, rows, cols)
    engine.mm_experts_dx(ty, w, off, dy, dx, 1024, n_row, rows, cols)
    torch.cuda.synchronize()
    assert torch.equal(y[:live].cpu(), (x64 @ w64.t()).to(t)) and (y[live:] == 77.0).all()
    assert torch.equal(dx[:live].cpu(), (dy64 @ w64).to(t)) and (dx[live:] == 77.0).all()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("rows,cols", [(2048, 2064), (2048, 2065), (32816, 128), (24, 175001)])
def test_weights_gradient_past_32_bits(engine, ty, rows, cols):
    """Gradients of 1024 experts, zeros but for the first and the last, which begins past 2^32 values."""
    import torch
    gen, t, live = torch.Generator().manual_seed(18), dtype(ty), 45
    assert 1023 * rows * cols > 1 << 32
    x, dy = whole(gen, live, cols), whole(gen, live, rows)
    off = torch.full((1025,), 5, dtype=torch.int32, device="cuda")
    off[0], off[1024] = 0, live
    dw = torch.full((1024, rows * cols), 77.0, dtype=t, device="cuda")
    engine.mm_experts_dw(ty, dy.to(t).cuda(), x.to(t).cuda(), off, dw, 1024, live, rows, cols)
    torch.cuda.synchronize()
    for e, s in ((0, slice(0, 5)), (1023, slice(5, live))):
        assert torch.equal(dw[e].cpu().reshape(rows, cols), (dy[s].t() @ x[s]).to(t)), e
    for e in range(1, 1023, 73):
        assert not dw[e:min(e + 73, 1023)].any(), e
