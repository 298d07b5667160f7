"""Expert routing, products and the way back run together, as an engine uses them, and under captured graphs, other streams and
workspaces of their own."""
import numpy as np
import pytest

import lastengine_amd as le
from tests.test_gpu_g4 import dequant, make
from tests.test_gpu_graphs import capture
from tests.test_gpu_route import route_plain, sort_plain
from tests.util import acts, weights

pytestmark = pytest.mark.gpu


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.mark.parametrize("n_tok", [1, 20, 300])
def test_steps_make_the_layer(engine, n_tok):
    """route -> sort -> grouped matmuls -> combine gives what le_moe_layer gives (both within the layer's parity bar of 1e-3 of
    the exact result, so within twice that of each other), with the same selection and the weights to fp32 rounding."""
    import torch
    tg, td, n_exp, k, hidden, ff = le.Q4_K, le.Q6_K, 16, 4, 1024, 512
    g, u, d = (dev(weights(ty, n_exp * r, c, 60 + i)[0]) for i, (ty, r, c) in enumerate(((tg, ff, hidden), (tg, ff, hidden), (td, hidden, ff))))
    h = dev(acts(n_tok * hidden, 70).reshape(n_tok, hidden))
    logits = dev(acts(n_tok * n_exp, 71).reshape(n_tok, n_exp))
    want = torch.empty(n_tok, hidden, device="cuda")
    li, lw = torch.empty(n_tok, k, dtype=torch.int32, device="cuda"), torch.empty(n_tok, k, device="cuda")
    engine.moe(tg, tg, td, g, u, d, n_exp, k, hidden, ff, logits, h, n_tok, want, idx_out=li, w_out=lw)
    n = n_tok * k
    idx, w = torch.empty_like(li), torch.empty_like(lw)
    off = torch.empty(n_exp + 1, dtype=torch.int32, device="cuda")
    i, o, pos = (torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(3))
    engine.moe_route(le.F32, logits, n_tok, n_exp, k, idx, w)
    engine.moe_sort(idx, n_tok, k, n_exp, off, i, o, pos)
    assert torch.equal(idx, li) and float((w - lw).abs().max()) <= 2e-6
    gate, up, down = torch.empty(n, ff, device="cuda"), torch.empty(n, ff, device="cuda"), torch.empty(n, hidden, device="cuda")
    engine.mm_grouped(tg, off, i, o, n_exp, n, h, gate, ff, hidden, w=g)
    engine.mm_grouped(tg, off, i, o, n_exp, n, h, up, ff, hidden, w=u)
    a = gate * torch.sigmoid(gate) * up
    engine.mm_grouped(td, off, o, o, n_exp, n, a, down, hidden, ff, w=d)
    out = torch.empty(n_tok, hidden, device="cuda")
    engine.moe_combine(le.F32, down, None, w, n_tok, k, hidden, out, n)  # rows in pair order
    assert float((out - want).abs().max()) <= 2e-3 * float(want.abs().max())
    # the same through rows in expert order: copied, multiplied in place order, brought back by pos
    rows, down2, out2 = torch.empty(n, hidden, device="cuda"), torch.empty(n, hidden, device="cuda"), torch.empty(n_tok, hidden, device="cuda")
    engine.moe_permute(le.F32, h, pos, n_tok, k, hidden, rows, n)
    place = torch.arange(n, dtype=torch.int32, device="cuda")
    engine.mm_grouped(tg, off, place, place, n_exp, n, rows, gate, ff, hidden, w=g)
    engine.mm_grouped(tg, off, place, place, n_exp, n, rows, up, ff, hidden, w=u)
    engine.mm_grouped(td, off, place, place, n_exp, n, gate * torch.sigmoid(gate) * up, down2, hidden, ff, w=d)
    engine.moe_combine(le.F32, down2, pos, w, n_tok, k, hidden, out2, n)
    assert torch.equal(out2, out)


@pytest.mark.parametrize("n_tok,pads", [(1, 1), (20, 3), (300, 40), (64, 64)])
def test_steps_with_padding(engine, n_tok, pads):
    """Padding tokens have no pairs: rows in place order and pos give them zeros whatever the rows' buffer held, and the others
    what the layer gives for them alone (twice the layer's parity bar)."""
    import torch
    tg, td, n_exp, k, hidden, ff = le.Q4_K, le.Q6_K, 16, 4, 256, 256
    g, u, d = (dev(weights(ty, n_exp * r, c, 80 + i)[0]) for i, (ty, r, c) in enumerate(((tg, ff, hidden), (tg, ff, hidden), (td, hidden, ff))))
    h = dev(acts(n_tok * hidden, 90).reshape(n_tok, hidden))
    logits = dev(acts(n_tok * n_exp, 91).reshape(n_tok, n_exp))
    live = n_tok - pads
    logits[live:] = -torch.inf
    n = n_tok * k
    idx, w = torch.empty(n_tok, k, dtype=torch.int32, device="cuda"), torch.empty(n_tok, k, device="cuda")
    off = torch.empty(n_exp + 1, dtype=torch.int32, device="cuda")
    i, o, pos = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(3))
    engine.moe_route(le.F32, logits, n_tok, n_exp, k, idx, w)
    engine.moe_sort(idx, n_tok, k, n_exp, off, i, o, pos)
    assert int(off[-1]) == live * k
    gate, up, down = (torch.full((n, c), float("nan"), device="cuda") for c in (ff, ff, hidden))
    place = torch.arange(n, dtype=torch.int32, device="cuda")
    engine.mm_grouped(tg, off, i, place, n_exp, n, h, gate, ff, hidden, w=g)
    engine.mm_grouped(tg, off, i, place, n_exp, n, h, up, ff, hidden, w=u)
    engine.mm_grouped(td, off, place, place, n_exp, n, gate * torch.sigmoid(gate) * up, down, hidden, ff, w=d)
    assert torch.isnan(down[live * k:]).all()
    out = torch.full((n_tok, hidden), float("nan"), device="cuda")
    engine.moe_combine(le.F32, down, pos, w, n_tok, k, hidden, out, n)
    assert (out[live:] == 0).all()
    if live:
        want = torch.empty(live, hidden, device="cuda")
        engine.moe(tg, tg, td, g, u, d, n_exp, k, hidden, ff, logits[:live], h[:live], live, want)
        assert float((out[:live] - want).abs().max()) <= 2e-3 * float(want.abs().max())


def g4_stack(n_mat, rows, cols, group, seed):
    codes, scales, z = make(n_mat, rows, cols, group, le.F16, True, seed)
    return le.G4(codes.cuda(), scales.cuda(), z.cuda(), rows, cols, group, n_mat=n_mat), dequant(codes, scales, z, group)[0]


class Decode:
    """A routed expert layer of 4-bit stacks at a few tokens: router, gate and up, SwiGLU and down, combine; the last token padding."""

    def __init__(self, ty, n_tok, seed):
        import torch
        self.ty, self.n_tok, self.n_exp, self.k, self.hidden, self.ff = ty, n_tok, 12, 3, 256, 160
        tt = {le.F32: torch.float32, le.F16: torch.float16, le.BF16: torch.bfloat16}[ty]
        self.gu, self.gu64 = g4_stack(self.n_exp, 2 * self.ff, self.hidden, 64, seed)
        self.dn, self.dn64 = g4_stack(self.n_exp, self.hidden, self.ff, 32, seed + 1)
        n = n_tok * self.k
        self.logits = torch.zeros(n_tok, self.n_exp, device="cuda")
        self.h = torch.zeros(n_tok, self.hidden, dtype=tt, device="cuda")
        self.idx, self.w = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, device="cuda")
        self.mid = torch.zeros(n, 2 * self.ff, dtype=tt, device="cuda")
        self.rows, self.out = torch.zeros(n, self.hidden, dtype=tt, device="cuda"), torch.zeros(n_tok, self.hidden, dtype=tt, device="cuda")

    def fill(self, seed):
        import torch
        g = torch.Generator().manual_seed(seed)
        l = torch.randn(self.n_tok, self.n_exp, generator=g)
        if self.n_tok > 1:
            l[-1] = -torch.inf
        self.logits.copy_(l)
        self.h.copy_(torch.randn(self.n_tok, self.hidden, generator=g))
        self.out.fill_(float("nan"))
        return l

    def run(self, engine, stream=None):
        n = self.n_tok * self.k
        engine.moe_route(le.F32, self.logits, self.n_tok, self.n_exp, self.k, self.idx, self.w, stream=stream)
        engine.mv_g4(self.ty, self.gu, self.h, self.mid, slots=n, share=self.k, sel=self.idx, stream=stream)
        engine.mv_g4(self.ty, self.dn, self.mid, self.rows, slots=n, sel=self.idx, swiglu=True, stream=stream)
        engine.moe_combine(self.ty, self.rows, None, self.w, self.n_tok, self.k, self.hidden, self.out, n, stream=stream)

    def check(self, l):
        import torch
        idx, w, _ = route_plain(l.double(), self.k)
        h, eps = self.h.double().cpu(), torch.finfo(self.out.dtype).eps
        want, mag = torch.zeros(self.n_tok, self.hidden, dtype=torch.float64), torch.zeros(self.n_tok, 1, dtype=torch.float64)
        for t in range(self.n_tok):
            for s in range(self.k):
                e = int(idx[t, s])
                if e < 0:
                    continue
                gu = self.gu64[e] @ h[t]
                y = self.dn64[e] @ (gu[:self.ff] / (1 + (-gu[:self.ff]).exp()) * gu[self.ff:])
                want[t] += w[t, s] * y
                mag[t] += w[t, s] * y.norm()
        # three roundings to the type on the way (gate and up, whose relative error SwiGLU makes at most twice as large in gate and
        # once in up, the rows, the sum): (2 + 1 + 1 + 1) eps / 2 of each row's norm, and fp32 sums far below
        err = (self.out.double().cpu() - want).norm(dim=1, keepdim=True)
        assert torch.isfinite(self.out).all() and (err <= 2.5 * eps * mag + 1e-4 * mag).all(), float((err / mag).max())
        if self.n_tok > 1:
            assert (self.out[-1] == 0).all()


@pytest.mark.parametrize("ty", [le.F32, le.F16, le.BF16])
@pytest.mark.parametrize("n_tok", [1, 5])
def test_decode_through_4_bit_experts(engine, ty, n_tok):
    d = Decode(ty, n_tok, 30)
    l = d.fill(1)
    d.run(engine)
    d.check(l)


def test_decode_graphs_side_by_side(engine):
    """Two captured layers replayed on two streams at once, several times, with new inputs and eager work between."""
    import torch
    ds = [Decode(le.F32, 4, 40), Decode(le.BF16, 3, 50)]
    graphs = [capture(lambda s, d=d: d.run(engine, s)) for d in ds]
    streams = [torch.cuda.Stream() for _ in ds]
    for rep in range(4):
        ls = [d.fill(100 + 10 * rep + i) for i, d in enumerate(ds)]
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for d, l in zip(ds, ls):
            d.check(l)
        l = ds[0].fill(500 + rep)  # the same buffers, eagerly
        ds[0].run(engine)
        ds[0].check(l)


class Train:
    """Sort, copies, weighted sum and every gradient of one step, with a workspace of its own."""

    def __init__(self, engine, n_tok, seed):
        import torch
        self.n_tok, self.k, self.n_exp, self.cols = n_tok, 4, 24, 200
        n = n_tok * self.k
        z = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
        self.logits, self.x, self.dout = z(n_tok, self.n_exp), z(n_tok, self.cols), z(n_tok, self.cols)
        self.idx, self.w = z(n, t=torch.int32), z(n)
        self.off, self.pos, self.i, self.o = z(self.n_exp + 1, t=torch.int32), z(n, t=torch.int32), z(n, t=torch.int32), z(n, t=torch.int32)
        self.rows, self.out = z(n, self.cols), z(n_tok, self.cols)
        self.drows, self.dw, self.dl, self.dx = z(n, self.cols), z(n), z(n_tok, self.n_exp), z(n_tok, self.cols)
        self.ws = z(max(16, engine.moe_sort_workspace_size(n_tok, self.k, self.n_exp)), t=torch.uint8)

    def fill(self, seed):
        import torch
        g = torch.Generator().manual_seed(seed)
        self.logits.copy_(torch.randn(self.logits.shape, generator=g))
        self.logits[-2:] = -torch.inf
        self.x.copy_(torch.randn(self.x.shape, generator=g))
        self.dout.copy_(torch.randn(self.dout.shape, generator=g))

    def run(self, eng, stream=None):
        n, k, e, c, r = self.n_tok, self.k, self.n_exp, self.cols, self.n_tok * self.k
        eng.moe_route(le.F32, self.logits, n, e, k, self.idx, self.w, stream=stream)
        eng.moe_sort(self.idx, n, k, e, self.off, self.i, self.o, self.pos, ws=self.ws, stream=stream)
        eng.moe_permute(le.F32, self.x, self.pos, n, k, c, self.rows, r, stream=stream)
        eng.moe_combine(le.F32, self.rows, self.pos, self.w, n, k, c, self.out, r, stream=stream)  # experts that pass their rows on
        eng.moe_combine_bwd(le.F32, self.dout, self.rows, self.pos, self.w, n, k, c, self.drows, self.dw, r, stream=stream)
        eng.moe_route_bwd(le.F32, self.idx, self.w, self.dw, n, e, k, self.dl, stream=stream)
        eng.moe_combine(le.F32, self.drows, self.pos, None, n, k, c, self.dx, r, stream=stream)

    def check(self):
        """Experts that pass their rows on: out = x (the weights sum to 1), dx = dout and dlogits = 0, to the roundings of sums of
        k terms (and, for dlogits, of the two sums of `cols` products that cancel: 2 (cols + k + 4) u of their magnitudes)."""
        import torch
        live = self.n_tok - 2
        idx = self.idx.reshape(self.n_tok, self.k).cpu().numpy()
        off, i, o, pos = sort_plain(idx, self.k, self.n_exp)
        assert np.array_equal(self.off.cpu().numpy(), off) and np.array_equal(self.pos.cpu().numpy(), pos)
        assert np.array_equal(self.i.cpu().numpy()[:len(i)], i) and np.array_equal(self.o.cpu().numpy()[:len(o)], o)
        u = 2.0 ** -24
        wi, ww, _ = route_plain(self.logits.double().cpu(), self.k)
        assert np.array_equal(idx, wi.numpy())
        x, dout = self.x.double(), self.dout.double()
        for got, want in ((self.out, x), (self.dx, dout)):
            assert ((got.double()[:live] - want[:live]).abs() <= 64 * u * want[:live].abs()).all() and (got[live:] == 0).all()
        mag = (x * dout).abs().sum(1, keepdim=True)
        assert (self.dl.double().abs()[:live] <= 4 * (self.cols + 8) * u * mag[:live]).all() and (self.dl[live:] == 0).all()
        want = (x * dout).sum(1, keepdim=True).expand(-1, self.k)[:live]
        assert ((self.dw.double().reshape(self.n_tok, self.k)[:live] - want).abs() <= (self.cols + 1) * u * mag[:live]).all()


@pytest.mark.parametrize("n_tok", [9, 3001])
def test_training_step(engine, n_tok):
    t = Train(engine, n_tok, 1)
    t.fill(7)
    t.run(engine)
    t.check()


def test_training_graphs_side_by_side(engine):
    """Two captured steps with workspaces of their own on two streams at once; replays with new inputs and eager steps between."""
    import torch
    ts = [Train(engine, 3001, 1), Train(engine, 2500, 2)]
    for t in ts:
        t.fill(1)
    graphs = [capture(lambda s, t=t: t.run(engine, s)) for t in ts]
    streams = [torch.cuda.Stream() for _ in ts]
    for rep in range(4):
        for i, t in enumerate(ts):
            t.fill(20 + 10 * rep + i)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for t in ts:
            t.check()
        ts[1].fill(300 + rep)
        ts[1].run(engine)
        torch.cuda.synchronize()
        ts[1].check()
