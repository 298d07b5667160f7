"""le_add_rms_quant against its definition, step by step in numpy: every output is the same to the bit (sum, 1 / sqrt and first product in 64
bits, where the order of a sum moves the result by some 2^-53 of it; a value that this carries over a rounding's border
would be one in 2^28, and the inputs are fixed)."""
import numpy as np
import pytest

import lastengine_amd as le
from tests.test_gpu_experts import TYPES, Rows, dtype
from tests.test_gpu_graphs import capture

pytestmark = pytest.mark.gpu


def reference(x, res, w, ty, eps, quantized=True):
    """x, res: tensors of type ty on the CPU -> h, o (fp32), xq, xd, xs."""
    import torch
    h = x if res is None else (x.float() + res.float()).to(dtype(ty))
    v = h.double().numpy()
    n = v.shape[1]
    with np.errstate(all="ignore"):
        s = (v * v).sum(1, keepdims=True)
        r = np.where(s < np.inf, 1.0 / np.sqrt(s / n + float(np.float32(eps))), np.nan)
        o = (v * r).astype(np.float32) * w.numpy()
        if not quantized:
            return h, torch.from_numpy(o), None, None, None
        u = o.reshape(len(v), n // 32, 32)
        d = np.abs(u).max(2) / np.float32(127.0)
        inv = np.where(d > 0, np.float32(1.0) / d, np.float32(0.0)).astype(np.float32)
        q = np.nan_to_num(np.clip(np.rint(u * inv[:, :, None]), -127, 127), nan=0.0).astype(np.int8)
    return h, torch.from_numpy(o), torch.from_numpy(q.reshape(len(v), n)), torch.from_numpy(d), torch.from_numpy(q.astype(np.int32).sum(2).astype(np.int32))


def same(got, want):
    """The same bits, NaN where NaN."""
    import torch
    return torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~torch.isnan(got)], want[~torch.isnan(want)])


class Case:
    def __init__(self, ty, m, n, seed, res=True, gap=0, at=0, size=1.0, h=True, o=True, q=True, xs=True, eps=1e-5):
        import torch
        gen = torch.Generator().manual_seed(seed)
        t = dtype(ty)
        self.ty, self.m, self.n, self.eps = ty, m, n, eps
        self.x, self.res = Rows(ty, m, n, n + gap, at), Rows(ty, m, n, n + gap, at) if res else None
        self.x.rows.copy_((torch.randn(m, n, generator=gen) * size).to(t))
        if res:
            self.res.rows.copy_((torch.randn(m, n, generator=gen) * size).to(t))
        self.wrows = Rows(le.F32, 1, n, None, at)
        self.wrows.rows.copy_(torch.randn(1, n, generator=gen) * 0.3 + 1.0)
        self.h, self.o = (Rows(ty, m, n, n + gap, at, 77.0) if wanted else None for wanted in (h, o))
        self.xq = torch.full((m * n + 64,), 99, dtype=torch.int8, device="cuda") if q else None
        self.xd = torch.full((m * (n // 32) + 64,), 77.0, device="cuda") if q else None
        self.xs = torch.full((m * (n // 32) + 64,), 777, dtype=torch.int32, device="cuda") if q and xs else None

    def run(self, engine, stream=None, h=None, m=None):
        h = h or self.h
        ptr = lambda r: r.ptr if r is not None else None  # noqa: E731
        ld = lambda r: r.stride if r is not None else 0  # noqa: E731
        engine.add_rms_quant(self.ty, self.x.ptr, ptr(self.res), self.wrows.ptr, ptr(h), ptr(self.o), self.xq, self.xd, self.xs, self.m, self.n, self.eps,
                             ldx=self.x.stride, ldr=ld(self.res), ldh=ld(h), ldo=ld(self.o), stream=stream)

    def want(self):
        return reference(self.x.rows.cpu(), self.res.rows.cpu() if self.res else None, self.wrows.rows[0].cpu(), self.ty, self.eps, self.xq is not None)

    def check(self, want=None, h=None):
        import torch
        torch.cuda.synchronize()
        wh, wo, wq, wd, ws = want or self.want()
        if h is None and self.h is not None:
            assert self.h.untouched(self.m, 77.0)
        h = h or self.h
        if h is not None:
            assert same(h.rows.cpu(), wh)
        if self.o is not None:
            assert same(self.o.rows.cpu(), wo.to(dtype(self.ty))) and self.o.untouched(self.m, 77.0) or torch.isnan(wo).any()
        if self.xq is not None:
            k = self.m * self.n
            assert same(self.xd[:k // 32].cpu(), wd.reshape(-1)) and (self.xd[k // 32:] == 77.0).all()
            assert torch.equal(self.xq[:k].cpu(), wq.reshape(-1)) and (self.xq[k:] == 99).all()
            if self.xs is not None:
                assert torch.equal(self.xs[:k // 32].cpu(), ws.reshape(-1)) and (self.xs[k // 32:] == 777).all()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("m,n", [(1, 32), (1, 4096), (3, 64), (37, 2048), (5, 96), (2, 5120), (300, 1056), (7, 8192), (2, 16416), (1, 40000), (1, 131072), (4099, 128)])
@pytest.mark.parametrize("res", [True, False])
def test_bits(engine, ty, m, n, res):
    c = Case(ty, m, n, 1, res=res)
    c.run(engine)
    c.check()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("m,n", [(1100, 384), (1100, 544), (300, 1536), (300, 2080), (300, 4128), (3, 8224), (2, 12320)])
def test_bits_of_every_shape_of_row(engine, ty, m, n):
    c = Case(ty, m, n, 7, xs=False)
    c.run(engine)
    c.check()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("gap,at", [(8, 0), (3, 0), (0, 1), (32, 8), (5, 3)])
@pytest.mark.parametrize("n", [64, 2080])
def test_strides_and_alignment(engine, ty, gap, at, n):
    c = Case(ty, 6, n, 2, gap=gap, at=at)
    c.run(engine)
    c.check()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("kw", [dict(h=False), dict(o=False), dict(xs=False), dict(h=False, o=False), dict(q=False), dict(q=False, h=False), dict(q=False, o=False, res=False)])
def test_outputs_left_out(engine, ty, kw):
    c = Case(ty, 9, 1024, 3, **kw)
    c.run(engine)
    c.check()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("n", [1, 7, 33, 100, 1001, 4097, 20001])
def test_norm_of_any_length(engine, ty, n):
    for gap, at in ((0, 0), (7, 1)):
        c = Case(ty, 5, n, 4, q=False, gap=gap, at=at)
        c.run(engine)
        c.check()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("n", [64, 4096, 40000])
def test_in_place(engine, ty, n):
    for kw in (dict(), dict(gap=8)):
        for where in ("x", "res"):
            c = Case(ty, 5, n, 5, h=False, **kw)
            want = c.want()
            target = getattr(c, where)
            c.run(engine, h=target)
            c.check(want, target)


@pytest.mark.parametrize("ty", TYPES)
def test_sizes_of_values(engine, ty):
    """Rows of the largest and of very small values, of zeros with and without eps."""
    big, little = {le.F32: (1e38, 1e-36), le.F16: (6e3, 1e-6), le.BF16: (1e38, 1e-36)}[ty]
    for size in (big, little):
        for eps in (1e-5, 0.0):
            c = Case(ty, 4, 512, 6, size=size / 4, eps=eps)
            c.run(engine)
            c.check()
    for eps in (1e-5, 0.0):
        c = Case(ty, 3, 256, 7, eps=eps)
        c.x.rows[1], c.res.rows[1] = 0.0, 0.0
        c.run(engine)
        want = list(c.want())
        if eps == 0.0:  # 0 / 0: not a number, and no codes
            want[2][1], want[4][1] = 0, 0
            want[3][1] = float("nan")
        c.check(want)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("n", [128, 4096, 40000])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_rows_that_are_not_finite(engine, ty, n, bad):
    import torch
    c = Case(ty, 6, n, 8)
    c.x.rows[2, n // 2] = bad
    c.run(engine)
    torch.cuda.synchronize()
    wh, wo, wq, wd, ws = c.want()
    assert same(c.h.rows.cpu(), wh)
    assert torch.isnan(c.o.rows[2]).all() and same(c.o.rows.cpu(), wo.to(dtype(ty)))
    xd, xq, xs = c.xd[:6 * n // 32].reshape(6, -1).cpu(), c.xq[:6 * n].reshape(6, -1).cpu(), c.xs[:6 * n // 32].reshape(6, -1).cpu()
    assert torch.isnan(xd[2]).all() and (xq[2] == 0).all() and (xs[2] == 0).all()
    rest = [0, 1, 3, 4, 5]
    assert torch.equal(xd[rest], wd[rest]) and torch.equal(xq[rest], wq[rest]) and torch.equal(xs[rest], ws[rest])


def test_far_rows(engine):
    import torch
    ld, n = (1 << 30) + 8, 64
    big = [torch.empty(4 * ld + n, dtype=torch.float16, device="cuda").as_strided((5, n), (ld, 1)) for _ in range(2)]
    x = torch.randn(5, n, generator=torch.Generator().manual_seed(9)).half()
    big[0].copy_(x)
    w = torch.ones(n, device="cuda")
    xq, xd = torch.empty(5, n, dtype=torch.int8, device="cuda"), torch.empty(5, n // 32, device="cuda")
    engine.add_rms_quant(le.F16, big[0], None, w, None, big[1], xq, xd, None, 5, n, 1e-6, ldx=ld, ldo=ld)
    _, wo, wq, wd, _ = reference(x, None, w.cpu(), le.F16, 1e-6)
    assert torch.equal(big[1].cpu(), wo.half()) and torch.equal(xq.cpu(), wq) and torch.equal(xd.cpu(), wd)


def test_what_the_other_entries_take(engine):
    """Of one fp32 row the norm is le_rms_quant's to fp32 rounding (its sum is in 32 bits), the int8 values are le_quant_x's of o, and
    le_matvec_q8 takes them."""
    import torch
    from tests.util import weights
    n, rows = 1024, 256
    c = Case(le.F32, 1, n, 10, res=False)
    c.run(engine)
    o, xq, xd, xs = torch.empty(n, device="cuda"), torch.empty(n, dtype=torch.int8, device="cuda"), torch.empty(n // 32, device="cuda"), torch.empty(n // 32, dtype=torch.int32, device="cuda")
    engine.rms_quant(c.x.rows[0].contiguous(), c.wrows.rows[0].contiguous(), o, xq, xd, xs, n, c.eps)
    mine = c.o.rows[0].contiguous()
    # le_rms_quant: a sum of n terms in 32 bits under a root, 1 / sqrt, two products; each step at most 2^-23
    assert ((o - mine).abs() <= (n / 2 + 8) * 2.0 ** -23 * mine.abs()).all()
    engine.quant_x(mine, xq, xd, xs, n // 32)
    torch.cuda.synchronize()
    assert torch.equal(xq, c.xq[:n]) and torch.equal(xd, c.xd[:n // 32]) and torch.equal(xs, c.xs[:n // 32])
    q = torch.from_numpy(weights(le.Q8_0, rows, n, 1)[0]).cuda()
    y, y2 = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    engine.mv_q8(le.Q8_0, None, c.xq, c.xd, c.xs, y, rows, n, 0, 1, w=q)
    engine.mv_q8(le.Q8_0, None, xq, xd, xs, y2, rows, n, 0, 1, w=q)
    torch.cuda.synchronize()
    assert torch.equal(y, y2) and float(y.abs().max()) > 0


def test_on_given_streams_and_in_graphs(engine):
    import torch
    cs = [Case(le.F32, 1, 4096, 11), Case(le.BF16, 50, 2048, 12)]
    graphs = [capture(lambda s, c=c: c.run(engine, s)) for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    for rep in range(4):
        for c in cs:
            c.x.rows.copy_(torch.randn(c.m, c.n, generator=torch.Generator().manual_seed(40 + rep)))
            c.o.flat.fill_(77.0)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for c in cs:
            c.check()
        cs[0].run(engine)
        cs[0].check()
    cs[1].o.flat.fill_(77.0)
    torch.cuda.synchronize()
    cs[1].run(engine, streams[0])
    cs[1].check()


def weights_of(c, w):
    c.wrows.rows.copy_(w)
    return c


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("m,n", [(3, 64), (2, 2080), (5, 4096), (1, 40000)])
@pytest.mark.parametrize("size", [1e-36, 1e-37, 3e-39, 1e-41, 1e-44])
def test_units_whose_scale_has_no_reciprocal(engine, ty, m, n, size):
    """The smallest fp32 weights: xd down to the last subnormal numbers and 0, with zeros in every unit and a unit of zeros."""
    import torch
    gen = torch.Generator().manual_seed(13)
    w = ((torch.randn(1, n, generator=gen).double() + 3.0) * size).float()
    w[0, ::5] = 0.0
    w[0, 32:64] = 0.0
    c = weights_of(Case(ty, m, n, 14), w)
    c.run(engine)
    h, o, _, d, _ = reference(c.x.rows.cpu(), c.res.rows.cpu(), w[0], ty, c.eps)
    u, far = o.numpy().reshape(m, n // 32, 32), d.numpy() < np.float32(2.0 ** -126)
    up = np.where(far, np.float32(2.0 ** 64), np.float32(1.0))
    with np.errstate(divide="ignore"):
        inv = np.where(d.numpy() > 0, np.float32(1.0) / (d.numpy() * up), np.float32(0.0)).astype(np.float32)
    q = np.clip(np.rint((u * up[:, :, None]) * inv[:, :, None]), -127, 127)
    # what the codes stand for: half a code from the quotient, a product and a reciprocal in 32 bits off by 2^-24 of up to 190 each (xd's own rounding, where it
    # has few bits, makes a quotient of up to 190, which is cut to 127)
    live = d.numpy() > 0
    ratio = np.clip(u.astype(np.float64)[live] / d.double().numpy()[live][:, None], -127.0, 127.0)
    assert (np.abs(q[live] - ratio) <= 0.5 + 190 * 2.0 ** -22).all() and (q[u == 0] == 0).all()
    q = q.astype(np.int8)
    c.check([h, o, torch.from_numpy(q.reshape(m, n)), d, torch.from_numpy(q.astype(np.int32).sum(2).astype(np.int32))])
    if size < 1e-37:
        assert far.all()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("m,n", [(3, 96), (2, 2080), (4, 4096), (1, 40000)])
def test_units_that_are_not_finite(engine, ty, m, n):
    """Weights that are not finite and products beyond fp32 reach their own units alone, which get no codes."""
    import torch
    gen = torch.Generator().manual_seed(15)
    w = torch.randn(1, n, generator=gen) * 0.3 + 1.0
    w[0, 5] = float("nan")
    w[0, 33] = float("inf")
    w[0, n - 1] = -3e38  # beyond fp32 for a norm of 1.2 and more, -infinity or infinity
    w[0, n - 3] = float("-inf") if n > 96 else 1.0
    c = weights_of(Case(ty, m, n, 16), w)
    c.x.rows[:, n - 1], c.res.rows[:, n - 1] = 8.0, 8.0
    c.run(engine)
    h, o, q, d, s = reference(c.x.rows.cpu(), c.res.rows.cpu(), w[0], ty, c.eps)
    torch.cuda.synchronize()
    assert torch.isnan(d[:, 0]).all() and torch.isinf(d[:, 1]).all() and torch.isinf(d[:, -1]).all()
    for u in (0, 1, -1):
        assert (q.reshape(m, -1, 32)[:, u] == 0).all() and (s.reshape(m, -1)[:, u] == 0).all()
    k = m * n
    assert same(c.h.rows.cpu(), h) and same(c.o.rows.cpu(), o.to(dtype(ty))) and c.o.untouched(m, 77.0)
    assert same(c.xd[:k // 32].cpu(), d.reshape(-1)) and torch.equal(c.xq[:k].cpu(), q.reshape(-1)) and torch.equal(c.xs[:k // 32].cpu(), s.reshape(-1))


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("n,gap,at", [(256, 0, 0), (256, 8, 0), (4096, 3, 1), (33, 0, 0), (40000, 0, 0)])
def test_rows_of_zeros_without_eps(engine, ty, n, gap, at):
    """NaN in the row of zeros, every other value of o and what lies around it as it has to be."""
    import torch
    c = Case(ty, 5, n, 17, eps=0.0, gap=gap, at=at, q=n % 32 == 0)
    for t in (1, 4):
        c.x.rows[t], c.res.rows[t] = 0.0, -0.0
    c.run(engine)
    torch.cuda.synchronize()
    wh, wo, wq, wd, ws = c.want()
    assert torch.isnan(wo[[1, 4]]).all() and not torch.isnan(wo[[0, 2, 3]]).any()
    assert same(c.o.rows.cpu(), wo.to(dtype(ty)))
    assert c.o.untouched(c.m, 77.0) and c.h.untouched(c.m, 77.0)
    assert same(c.h.rows.cpu(), wh)
    if c.xq is not None:
        wq[[1, 4]], ws[[1, 4]], wd[[1, 4]] = 0, 0, float("nan")
        k = c.m * n
        assert torch.equal(c.xq[:k].cpu(), wq.reshape(-1)) and torch.equal(c.xs[:k // 32].cpu(), ws.reshape(-1)) and same(c.xd[:k // 32].cpu(), wd.reshape(-1))
