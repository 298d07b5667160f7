"""le_lora against the formula in 64 bits: whole numbers, whose sums fp32 holds exactly, so that every result has to be the exact one
rounded once; and real numbers within the bound of fp32 sums."""
import pytest

import lastengine_amd as le
from tests.test_gpu_experts import TYPES, Rows, dtype, half_step, real
from tests.test_gpu_graphs import capture

pytestmark = pytest.mark.gpu


def small(gen, *shape):
    import torch
    return torch.randint(-2, 3, shape, generator=gen, dtype=torch.float64)


def runs(gen, m, n_ad, each, bare):
    """Adapters of m tokens in runs of about `each`; a share of the runs has none."""
    import torch
    which = torch.randint(0, n_ad, (m,), generator=gen, dtype=torch.int32)
    which = torch.where(torch.rand(m, generator=gen) < bare, -1, which)
    return which[torch.arange(m) // each]


class Case:
    def __init__(self, xty, wty, m, rows, cols, rank, n_ad, seed, make=small, each=1, bare=0.2, base=True, gap=0, at=0, shared=False, scale=True):
        import torch
        gen = torch.Generator().manual_seed(seed)
        self.xty, self.m, self.rows, self.cols, self.rank, self.n_ad = xty, m, rows, cols, rank, n_ad
        xt, wt = dtype(xty), dtype(wty)
        self.x64 = make(gen, 1 if shared else m, cols).to(xt).double()
        self.a64, self.b64 = make(gen, n_ad, rank, cols).to(wt).double(), make(gen, n_ad, rows, rank).to(wt).double()
        self.s64 = torch.tensor([0.5, 1.0, 2.0, -1.0])[torch.randint(0, 4, (n_ad,), generator=gen)].double() if scale else torch.ones(n_ad).double()
        self.base64 = make(gen, m, rows).to(xt).double() if base else torch.zeros(m, rows).double()
        self.idx = runs(gen, m, n_ad, each, bare)
        self.x, self.base, self.y = Rows(xty, len(self.x64), cols, cols + gap, at), Rows(xty, m, rows, rows + gap, at), Rows(xty, m, rows, rows + gap, at, 77.0)
        self.x.rows.copy_(self.x64)
        self.base.rows.copy_(self.base64)
        self.a, self.b = Rows(wty, n_ad, rank * cols, None, at), Rows(wty, n_ad, rows * rank, None, at)
        self.a.rows.copy_(self.a64.reshape(n_ad, -1))
        self.b.rows.copy_(self.b64.reshape(n_ad, -1))
        self.scale = self.s64.float().cuda() if scale else None
        self.dev_idx = self.idx.cuda()
        self.has_base, self.ldx = base, 0 if shared else self.x.stride
        self.ad = le.Adapters(self.a.ptr, self.b.ptr, self.scale, n_ad, rank, rows, cols, ltype=wty)

    def run(self, engine, stream=None, ws=None, in_place=False):
        y = self.base if in_place else self.y
        engine.lora(self.xty, self.ad, self.dev_idx, self.x.ptr, self.base.ptr if self.has_base else None, y.ptr, self.m, ldx=self.ldx, ldb=self.base.stride,
                    ldy=y.stride, ws=ws, stream=stream)

    def want(self, f=lambda v: v):
        import torch
        y = f(self.base64).clone()
        x = f(self.x64).expand(self.m, -1)
        for i in range(self.n_ad):
            t = torch.nonzero(self.idx == i).reshape(-1)
            if len(t):
                y[t] += f(self.s64[i]) * ((x[t] @ f(self.a64[i]).t()) @ f(self.b64[i]).t())
        return y

    def check_whole(self, rows=None):
        import torch
        torch.cuda.synchronize()
        got = self.y if rows is None else rows
        if rows is None:
            assert self.y.untouched(self.m, 77.0)
        assert torch.equal(got.rows.cpu(), self.want().to(dtype(self.xty)))

    def check_real(self):
        """fp32 sums of cols, then of rank terms, a product with scale and a sum with base, each off by at most a last place (2^-23);
        then one rounding."""
        import torch
        torch.cuda.synchronize()
        want, mag = self.want(), self.want(torch.abs)
        bound = (self.cols + self.rank + 4) * 2.0 ** -23 * mag
        bound = bound + half_step(self.xty) * (want.abs() + bound) + (2.0 ** -25 if self.xty == le.F16 else 1e-38)
        assert ((self.y.rows.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("xty", TYPES)
@pytest.mark.parametrize("wty", TYPES)
@pytest.mark.parametrize("m,rows,cols,rank,n_ad,each", [
    (1, 256, 512, 16, 3, 1), (1, 1, 1, 1, 1, 1), (2, 33, 77, 5, 2, 1), (15, 200, 264, 12, 6, 5), (61, 520, 256, 16, 40, 1), (64, 64, 1032, 64, 4, 16), (70, 130, 96, 100, 3, 35),
    (200, 96, 160, 8, 9, 1), (300, 264, 320, 32, 5, 70), (129, 72, 40, 256, 2, 64), (40, 50, 515, 31, 7, 3), (513, 140, 136, 4, 70, 2), (300, 264, 320, 64, 5, 40), (257, 130, 96, 100, 3, 35), (700, 200, 72, 24, 6, 1)])
def test_whole_numbers(engine, xty, wty, m, rows, cols, rank, n_ad, each):
    c = Case(xty, wty, m, rows, cols, rank, n_ad, 1, each=each)
    c.run(engine)
    c.check_whole()


@pytest.mark.parametrize("xty", TYPES)
@pytest.mark.parametrize("m", [1, 9, 100, 300])
@pytest.mark.parametrize("kw", [dict(gap=8), dict(gap=3), dict(at=1), dict(gap=16, at=8), dict(base=False), dict(shared=True), dict(scale=False), dict(bare=1.0), dict(bare=0.0, each=1000)])
def test_forms(engine, xty, m, kw):
    """Rows apart and at odd addresses, no base, one row of x for all, no factors, no token or every token of one adapter."""
    for wty in (xty, le.BF16):
        c = Case(xty, wty, m, 96, 264, 16, 4, 2, **kw)
        c.run(engine)
        c.check_whole()


@pytest.mark.parametrize("xty", TYPES)
@pytest.mark.parametrize("m", [1, 20, 90, 261])
def test_in_place(engine, xty, m):
    c = Case(xty, xty, m, 200, 128, 8, 3, 3)
    c.run(engine, in_place=True)
    c.check_whole(c.base)


@pytest.mark.parametrize("xty", TYPES)
@pytest.mark.parametrize("wty", TYPES)
@pytest.mark.parametrize("m,rows,cols,rank,n_ad,each", [(1, 512, 4096, 16, 2, 1), (33, 300, 2048, 12, 8, 1), (260, 256, 1024, 64, 3, 100)])
def test_real_numbers(engine, xty, wty, m, rows, cols, rank, n_ad, each):
    c = Case(xty, wty, m, rows, cols, rank, n_ad, 4, make=real, each=each)
    c.run(engine)
    c.check_real()


def test_long_rows(engine):
    for xty in TYPES:
        c = Case(xty, xty, 3, 30000, 28672, 4, 2, 5, bare=0.0)
        c.run(engine)
        c.check_whole()


@pytest.mark.parametrize("xty", TYPES)
@pytest.mark.parametrize("m", [3, 50, 140, 270])
def test_what_is_not_finite_stays_with_its_token(engine, xty, m):
    """NaN in one adapter and infinity in one row of x: no token but theirs is touched, in a batch where the adapters alternate."""
    import torch
    c = Case(xty, xty, m, 72, 136, 8, 3, 6, bare=0.0)
    c.idx = (torch.arange(m) % 3).to(torch.int32)
    c.dev_idx.copy_(c.idx)
    want = c.want().to(dtype(xty))
    c.a.rows[1] = float("nan")
    c.b.rows[1] = float("inf")
    c.x.rows[2, 5] = float("inf")
    c.run(engine)
    torch.cuda.synchronize()
    got = c.y.rows.cpu()
    for t in range(m):
        if t == 2:
            continue
        assert not torch.isfinite(got[t]).any() if t % 3 == 1 else torch.equal(got[t], want[t]), t


@pytest.mark.parametrize("m", [4, 80, 260])
def test_numbers_of_no_adapter(engine, m):
    import torch
    c = Case(le.F32, le.F16, m, 64, 128, 8, 3, 7)
    c.idx[:4] = torch.tensor([-1, 3, 2**31 - 1, -2**31])
    c.dev_idx.copy_(c.idx)
    c.run(engine)
    c.check_whole()
    assert torch.equal(c.y.rows[:4], c.base.rows[:4])


def test_far_rows(engine):
    """x, base and y rows more than 2^32 values apart."""
    import torch
    gen = torch.Generator().manual_seed(8)
    m, rows, cols, rank, ld = 6, 24, 40, 4, (1 << 30) + 8
    big = [torch.empty(5 * ld + 64, dtype=torch.bfloat16, device="cuda").as_strided((m, c), (ld, 1)) for c in (cols, rows)]
    x, a, b = small(gen, m, cols), small(gen, 2, rank, cols), small(gen, 2, rows, rank)
    base = small(gen, m, rows)
    big[0].copy_(x)
    big[1].copy_(base)
    ad = le.Adapters(a.bfloat16().cuda(), b.bfloat16().cuda(), None, 2, rank, rows, cols)
    idx = torch.tensor([0, 1, 0, 1, 1, 0], dtype=torch.int32)
    engine.lora(le.BF16, ad, idx.cuda(), big[0], big[1], big[1], m, ldx=ld, ldb=ld, ldy=ld)
    want = torch.stack([base[t] + b[i] @ (a[i] @ x[t]) for t, i in enumerate(idx.tolist())])
    assert torch.equal(big[1].cpu(), want.bfloat16())


@pytest.mark.parametrize("m", [1, 30, 150, 400])
def test_same_bits_whatever_the_workspace_held(engine, m):
    import torch
    c = Case(le.F32, le.BF16, m, 300, 2048, 16, 5, 9, make=real)
    c.run(engine)
    torch.cuda.synchronize()
    first = c.y.rows.clone()
    n = engine.lora_workspace_size(le.F32, c.ad, m)
    for byte in (0, 255, 127):
        c.run(engine, ws=torch.full((n,), byte, dtype=torch.uint8, device="cuda"))
        torch.cuda.synchronize()
        assert torch.equal(c.y.rows, first)


def test_on_given_streams_and_in_graphs(engine):
    """Two captured calls with workspaces of their own, replayed on two streams at once with new inputs and other adapters, eager calls
    between; then an eager call on a stream."""
    import torch
    cs = [Case(le.F32, le.F16, 1, 256, 512, 16, 4, 10), Case(le.BF16, le.BF16, 200, 136, 264, 8, 6, 11, each=20)]
    wss = [torch.empty(engine.lora_workspace_size(c.xty, c.ad, c.m), dtype=torch.uint8, device="cuda") for c in cs]
    graphs = [capture(lambda s, c=c, ws=ws: c.run(engine, s, ws)) for c, ws in zip(cs, wss)]
    streams = [torch.cuda.Stream() for _ in cs]
    for rep in range(4):
        for c in cs:
            gen = torch.Generator().manual_seed(30 + rep)
            c.x64 = small(gen, *c.x64.shape)
            c.x.rows.copy_(c.x64)
            c.idx = runs(gen, c.m, c.n_ad, 1 + 7 * rep, 0.1)
            c.dev_idx.copy_(c.idx)
            c.y.flat.fill_(77.0)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for c in cs:
            c.check_whole()
        cs[1].run(engine)
        cs[1].check_whole()
    cs[0].y.flat.fill_(77.0)
    torch.cuda.synchronize()
    cs[0].run(engine, streams[1])
    cs[0].check_whole()


@pytest.mark.parametrize("ty", [le.Q4_K, le.Q8_0])
def test_beside_a_quantized_projection(engine, ty):
    """The projection of a batch by le_gemm with adapters added in place: what the two give apart, added."""
    import torch
    from tests.util import weights
    m, rows, cols = 20, 256, 512
    q = torch.from_numpy(weights(ty, rows, cols, 1)[0]).cuda()
    c = Case(le.F32, le.F16, m, rows, cols, 16, 4, 12, make=real)
    y = torch.empty(m, rows, device="cuda")
    engine.gemm(ty, q, c.x.ptr, m, y, rows, cols)
    c.base.rows.copy_(y)
    c.base64 = y.cpu().double()
    c.run(engine)
    c.check_real()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("m", [1, 20, 256, 257, 700])
def test_base_of_no_adapter_to_the_bit(engine, ty, m):
    """Zeros of both signs, infinities and the smallest values of base where there is no adapter; without a base zeros."""
    import torch
    t = dtype(ty)
    values = torch.tensor([-0.0, 0.0, float("inf"), -float("inf"), torch.finfo(t).smallest_normal / 4, -torch.finfo(t).max], dtype=t)
    for rows in (96, 99):
        c = Case(ty, ty, m, rows, 64, 8, 3, 13, bare=0.0)
        c.idx[::3] = -1
        c.dev_idx.copy_(c.idx)
        base = values[torch.arange(m * rows).reshape(m, rows) % len(values)]
        c.base.rows.copy_(base)
        bits = torch.int32 if ty == le.F32 else torch.int16
        for has_base in (True, False):
            c.has_base = has_base
            c.run(engine)
            torch.cuda.synchronize()
            want = base[::3] if has_base else torch.zeros_like(base[::3])
            assert torch.equal(c.y.rows.cpu()[::3].contiguous().view(bits), want.contiguous().view(bits))


@pytest.mark.parametrize("xty", [le.F32, le.BF16])
@pytest.mark.parametrize("wty", TYPES)
@pytest.mark.parametrize("m", [20, 256, 257, 400])
@pytest.mark.parametrize("rank", [16, 64, 100])
def test_far_factors(engine, xty, wty, m, rank):
    """Factors whose products with A x alone would leave fp32, though y does not. Powers of two, one rank live: exact."""
    import torch
    for scale, xs, bs in ((2.0 ** 100, 2.0 ** 40, 2.0 ** -14), (2.0 ** -120, 2.0 ** -20, 2.0 ** 14)):
        c = Case(xty, wty, m, 72, 64, rank, 3, 14, bare=0.0, base=False, scale=False)
        c.x64 = torch.zeros(m, 64).double()
        c.x64[:, 5] = xs * (1 + torch.arange(m) % 2)
        c.a64 = torch.zeros(3, rank, 64).double()
        c.a64[:, rank - 3] = 1.0
        c.b64 = torch.zeros(3, 72, rank).double()
        c.b64[:, :, rank - 3] = bs * (torch.arange(72) % 3 - 1).double()
        c.s64 = torch.full((3,), scale).double()
        c.x.rows.copy_(c.x64)
        c.a.rows.copy_(c.a64.reshape(3, -1))
        c.b.rows.copy_(c.b64.reshape(3, -1))
        c.scale = c.s64.float().cuda()
        c.ad = le.Adapters(c.a.ptr, c.b.ptr, c.scale, 3, rank, 72, 64, ltype=wty)
        c.run(engine)
        c.check_whole()
        assert float(c.y.rows.abs().max()) == 2 * scale * xs * bs


@pytest.mark.parametrize("xty,wty", [(x, w) for x in TYPES for w in TYPES if x != w])
@pytest.mark.parametrize("m", [3, 50, 140, 270])
def test_what_is_not_finite_stays_with_its_token_beside_another_type(engine, xty, wty, m):
    import torch
    c = Case(xty, wty, m, 72, 136, 8, 3, 15, bare=0.0)
    c.idx = (torch.arange(m) % 3).to(torch.int32)
    c.dev_idx.copy_(c.idx)
    want = c.want().to(dtype(xty))
    c.a.rows[1] = float("nan")
    c.b.rows[1] = float("inf")
    c.x.rows[2, 5] = float("inf")
    c.a.rows[2] += 10.0  # no zeros, so that all of token 2 is infinite or NaN
    c.b.rows[2, 3 * 8:] = 1.0
    c.b.rows[2, :3 * 8] = 0.0
    c.run(engine)
    torch.cuda.synchronize()
    got = c.y.rows.cpu()
    for t in range(m):
        if t == 2:
            assert not torch.isfinite(got[t, 3:]).any()
        elif t % 3 == 1:
            assert not torch.isfinite(got[t]).any()
        elif t % 3 == 0:
            assert torch.equal(got[t], want[t]), t
        else:
            assert torch.isfinite(got[t]).all(), t


@pytest.mark.parametrize("xty,wty", [(le.F32, le.F16), (le.F32, le.BF16), (le.F16, le.F32), (le.BF16, le.F32)])
@pytest.mark.parametrize("m", [20, 300])
@pytest.mark.parametrize("e", [-90, -108, -120, -128])
def test_small_fp32_beside_16_bits(engine, xty, wty, m, e):
    """The fp32 side's values around 2^e, the other's 2^up, brought near 1 by the second product and the factor: fp32 sums, and each value cut at 2^-133."""
    import torch
    gen = torch.Generator().manual_seed(16)
    cols, up = 64, 14
    c = Case(xty, wty, m, 40, cols, 16, 2, 17, bare=0.0, base=False)
    tiny = lambda *shape: ((1 + torch.rand(*shape, generator=gen, dtype=torch.float64)) * 2.0 ** e).float().double()  # noqa: E731
    c.x64 = tiny(m, cols) if xty == le.F32 else torch.full((m, cols), 2.0 ** up).double()
    c.a64 = tiny(2, 16, cols) if wty == le.F32 else torch.full((2, 16, cols), 2.0 ** up).double()
    c.b64 = torch.zeros(2, 40, 16).double()
    c.b64[:, torch.arange(40), torch.arange(40) % 16] = 2.0 ** 14
    c.s64 = torch.full((2,), 2.0 ** (-e - up - 14 - 6)).double()
    c.x.rows.copy_(c.x64)
    c.a.rows.copy_(c.a64.reshape(2, -1))
    c.b.rows.copy_(c.b64.reshape(2, -1))
    c.scale = c.s64.float().cuda()
    c.ad = le.Adapters(c.a.ptr, c.b.ptr, c.scale, 2, 16, 40, cols, ltype=wty)
    c.run(engine)
    torch.cuda.synchronize()
    want, total = c.want(), 2.0 ** (-e - up - 6)
    # the sums over cols and rank (cols + 16 steps and the factor), what is cut of the cols values and of their sum, one rounding
    bound = (cols + 20) * 2.0 ** -23 * want + (cols * 2.0 ** (-133 + up) + 2.0 ** -133) * total
    bound = bound + half_step(xty) * (want + bound) + (2.0 ** -25 if xty == le.F16 else 1e-38)
    assert float(want.min()) > 0.5 and ((c.y.rows.cpu().double() - want).abs() <= bound).all()
