"""The operators around the shared products run together, as an engine uses them: residual, norm and int8 activations, a quantized projection with
adapters beside it, routing, the experts' products and the way back; and a training step of the routed block with all its gradients."""
import pytest

import lastengine_amd as le
from tests.test_gpu_experts import dtype
from tests.test_gpu_graphs import capture
from tests.util import weights

pytestmark = pytest.mark.gpu


def z(*s, t=None):
    import torch
    return torch.zeros(*s, dtype=t or torch.float32, device="cuda")


class Serve:
    """One layer's step for a batch of requests, fp32: out = h + W o + adapter(o) + routed block(o)."""
    eps = 1e-5

    def __init__(self, engine, n, seed):
        import torch
        g = torch.Generator().manual_seed(seed)
        self.n, self.hidden, self.ff, self.e, self.k, self.rank, self.n_ad = n, 256, 96, 12, 3, 8, 4
        r = lambda *s, std=1.0: torch.randn(*s, generator=g) * std  # noqa: E731
        self.norm_w = (1.0 + r(self.hidden, std=0.1)).cuda()
        q = weights(le.Q8_0, self.hidden, self.hidden, seed, std=0.06)[0]
        self.q = torch.from_numpy(q).cuda()
        self.wq = z(self.hidden, self.hidden)
        engine.dequant_rows(le.Q8_0, self.q, self.wq, self.hidden, self.hidden)
        self.a, self.b = r(self.n_ad, self.rank, self.hidden, std=0.06).cuda(), r(self.n_ad, self.hidden, self.rank, std=0.3).cuda()
        self.scale = torch.tensor([0.5, 1.0, 2.0, -1.0]).cuda()
        self.ad = le.Adapters(self.a, self.b, self.scale, self.n_ad, self.rank, self.hidden, self.hidden)
        self.router = r(self.e, self.hidden, std=0.06).cuda()
        self.gu, self.down = r(self.e, 2 * self.ff, self.hidden, std=0.06).cuda(), r(self.e, self.hidden, self.ff, std=0.1).cuda()
        p = n * self.k
        self.x, self.res, self.who = z(n, self.hidden), z(n, self.hidden), z(n, t=torch.int32)
        self.h, self.o, self.xq, self.xd = z(n, self.hidden), z(n, self.hidden), z(n, self.hidden, t=torch.int8), z(n, self.hidden // 32)
        self.y, self.y8 = z(n, self.hidden), z(n, self.hidden)
        self.logits, self.idx, self.w = z(n, self.e), z(p, t=torch.int32), z(p)
        self.off, self.pos = z(self.e + 1, t=torch.int32), z(p, t=torch.int32)
        self.rows, self.mid, self.act, self.back, self.moe = z(p, self.hidden), z(p, 2 * self.ff), z(p, self.ff), z(p, self.hidden), z(n, self.hidden)
        self.ws = [z(max(16, s), t=torch.uint8) for s in (engine.gemm_workspace_size_rows(le.Q8_0, n, self.hidden, self.hidden),
                                                          engine.lora_workspace_size(le.F32, self.ad, n), engine.moe_sort_workspace_size(n, self.k, self.e))]
        self.out = z(n, self.hidden)

    def fill(self, seed):
        import torch
        g = torch.Generator().manual_seed(seed)
        self.x.copy_(torch.randn(self.x.shape, generator=g))
        self.res.copy_(torch.randn(self.x.shape, generator=g))
        self.who.copy_(torch.randint(-1, self.n_ad, (self.n,), generator=g))
        for t in (self.out, self.rows, self.mid, self.back):
            t.fill_(float("nan"))

    def run(self, eng, stream=None):
        import torch
        n, H, F, p, f32 = self.n, self.hidden, self.ff, self.n * self.k, le.F32
        kw = dict(stream=stream)
        eng.add_rms_quant(f32, self.x, self.res, self.norm_w, self.h, self.o, self.xq, self.xd, None, n, H, self.eps, **kw)
        eng.mv_q8(le.Q8_0, None, self.xq, self.xd, None, self.y8, H, H, 0, 1, w=self.q, **kw)  # the first token's int8 form
        if n > 1:
            eng.gemm(le.Q8_0, self.q, self.o, n, self.y, H, H, ws=self.ws[0], **kw)
        else:
            eng.mv(le.Q8_0, self.q, self.o, self.y, H, H, **kw)
        eng.lora(f32, self.ad, self.who, self.o, self.y, self.y, n, ws=self.ws[1], **kw)
        torch.matmul(self.o, self.router.t(), out=self.logits)
        eng.moe_route(f32, self.logits, n, self.e, self.k, self.idx, self.w, **kw)
        eng.moe_sort(self.idx, n, self.k, self.e, self.off, None, None, self.pos, ws=self.ws[2], **kw)
        eng.moe_permute(f32, self.o, self.pos, n, self.k, H, self.rows, p, **kw)
        eng.mm_experts(f32, self.gu, self.off, self.rows, self.mid, self.e, p, 2 * F, H, **kw)
        torch.mul(torch.nn.functional.silu(self.mid[:, :F]), self.mid[:, F:], out=self.act)
        eng.mm_experts(f32, self.down, self.off, self.act, self.back, self.e, p, H, F, **kw)
        eng.moe_combine(f32, self.back, self.pos, self.w, n, self.k, H, self.moe, p, **kw)
        torch.add(self.h, self.y, out=self.out)
        self.out.add_(self.moe)

    def check(self):
        """The parity bar of the quantized products (1e-3 of the largest value); the int8 form has an activation error of half
        a step of 1/127 of its unit's largest value, at most 2^-8 of it, on top, in 256 terms of random sign."""
        import torch
        torch.cuda.synchronize()
        d = lambda t: t.double().cpu()  # noqa: E731
        h = d(self.x) + d(self.res)
        o = h / torch.sqrt((h * h).mean(1, keepdim=True) + self.eps) * d(self.norm_w)
        y = o @ d(self.wq).t()
        y8 = y[0].clone()
        who = self.who.cpu()
        for i in range(self.n_ad):
            t = who == i
            y[t] += float(self.scale[i]) * (o[t] @ d(self.a[i]).t()) @ d(self.b[i]).t()
        idx, w = self.idx.cpu().long().reshape(self.n, self.k), d(self.w).reshape(self.n, self.k)
        logits = o @ d(self.router).t()
        assert (logits.gather(1, idx) >= logits.topk(self.k).values[:, -1:] - 1e-4).all()
        assert ((w - torch.softmax(logits.gather(1, idx), 1)).abs() <= 1e-4).all()
        moe = torch.zeros_like(h)
        for s in range(self.k):
            m = torch.einsum("nh,nfh->nf", o, d(self.gu)[idx[:, s]])
            a = m[:, :self.ff] * torch.sigmoid(m[:, :self.ff]) * m[:, self.ff:]
            moe += w[:, s:s + 1] * torch.einsum("nf,nhf->nh", a, d(self.down)[idx[:, s]])
        want = h + y + moe
        assert float((d(self.out) - want).abs().max()) <= 1e-3 * float(want.abs().max())
        assert float((d(self.y8[0]) - y8).abs().max()) <= (1e-3 + 2.0 ** -8) * float((o[0].abs() @ d(self.wq).abs().t()).max())


@pytest.mark.parametrize("n", [1, 6, 70, 300])
def test_layer(engine, n):
    s = Serve(engine, n, 1)
    s.fill(2)
    s.run(engine)
    s.check()


def test_layer_graphs_side_by_side(engine):
    """Two captured layers replayed on two streams at once, with new inputs and adapters, eager steps between."""
    import torch
    ss = [Serve(engine, 5, 3), Serve(engine, 90, 4)]
    for s in ss:
        s.fill(5)
    graphs = [capture(lambda st, s=s: s.run(engine, st)) for s in ss]
    streams = [torch.cuda.Stream() for _ in ss]
    for rep in range(4):
        for i, s in enumerate(ss):
            s.fill(10 * rep + i)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for s in ss:
            s.check()
        ss[0].fill(100 + rep)
        ss[0].run(engine)
        ss[0].check()


class Train:
    """The routed block and every gradient of it; the last tokens are padding."""

    def __init__(self, engine, ty, n, seed, hidden=64, ff=40, pads=2):
        import torch
        g = torch.Generator().manual_seed(seed)
        self.ty, self.n, self.live, self.hidden, self.ff, self.e, self.k = ty, n, n - pads, hidden, ff, 6, 2
        t, p = dtype(ty), n * self.k
        self.gu = (torch.randn(self.e, 2 * ff, hidden, generator=g) * hidden ** -0.5).to(t).cuda()
        self.down = (torch.randn(self.e, hidden, ff, generator=g) * ff ** -0.5).to(t).cuda()
        self.x, self.dout, self.logits = z(n, hidden, t=t), z(n, hidden, t=t), z(n, self.e)
        self.idx, self.w, self.off, self.pos = z(p, t=torch.int32), z(p), z(self.e + 1, t=torch.int32), z(p, t=torch.int32)
        self.rows, self.mid, self.act, self.back, self.out = z(p, hidden, t=t), z(p, 2 * ff, t=t), z(p, ff, t=t), z(p, hidden, t=t), z(n, hidden, t=t)
        self.dback, self.dw, self.dact, self.dmid, self.drows = z(p, hidden, t=t), z(p), z(p, ff, t=t), z(p, 2 * ff, t=t), z(p, hidden, t=t)
        self.ddown, self.dgu, self.dlogits, self.dx = z(self.e, hidden, ff), z(self.e, 2 * ff, hidden), z(n, self.e), z(n, hidden, t=t)
        self.ws = z(max(16, engine.moe_sort_workspace_size(n, self.k, self.e)), t=torch.uint8)
        self.wg = [z(max(16, engine.mm_experts_dw_workspace_size(ty, self.e, p, r, c)), t=torch.uint8) for r, c in ((hidden, ff), (2 * ff, hidden))]

    def fill(self, seed):
        import torch
        g = torch.Generator().manual_seed(seed)
        self.x.copy_(torch.randn(self.x.shape, generator=g))
        self.dout.copy_(torch.randn(self.dout.shape, generator=g))
        self.logits.copy_(torch.randn(self.logits.shape, generator=g))
        self.logits[self.live:] = -torch.inf
        for t in (self.out, self.dx, self.dgu, self.ddown, self.dlogits):
            t.fill_(float("nan"))

    def run(self, eng, stream=None):
        import torch
        n, H, F, e, k, p, ty, kw = self.n, self.hidden, self.ff, self.e, self.k, self.n * self.k, self.ty, dict(stream=stream)
        eng.moe_route(le.F32, self.logits, n, e, k, self.idx, self.w, **kw)
        eng.moe_sort(self.idx, n, k, e, self.off, None, None, self.pos, ws=self.ws, **kw)
        eng.moe_permute(ty, self.x, self.pos, n, k, H, self.rows, p, **kw)
        eng.mm_experts(ty, self.gu, self.off, self.rows, self.mid, e, p, 2 * F, H, **kw)
        gate, up = self.mid[:, :F].float(), self.mid[:, F:].float()
        sig = torch.sigmoid(gate)
        self.act.copy_(gate * sig * up)
        eng.mm_experts(ty, self.down, self.off, self.act, self.back, e, p, H, F, **kw)
        eng.moe_combine(ty, self.back, self.pos, self.w, n, k, H, self.out, p, **kw)
        eng.moe_combine_bwd(ty, self.dout, self.back, self.pos, self.w, n, k, H, self.dback, self.dw, p, **kw)
        eng.moe_route_bwd(le.F32, self.idx, self.w, self.dw, n, e, k, self.dlogits, **kw)
        eng.mm_experts_dw(ty, self.dback, self.act, self.off, self.ddown, e, p, H, F, dw_ty=le.F32, ws=self.wg[0], **kw)
        eng.mm_experts_dx(ty, self.down, self.off, self.dback, self.dact, e, p, H, F, **kw)
        da = self.dact.float()
        self.dmid[:, :F] = da * up * sig * (1 + gate * (1 - sig))
        self.dmid[:, F:] = da * gate * sig
        eng.mm_experts_dw(ty, self.dmid, self.rows, self.off, self.dgu, e, p, 2 * F, H, dw_ty=le.F32, ws=self.wg[1], **kw)
        eng.mm_experts_dx(ty, self.gu, self.off, self.dmid, self.drows, e, p, 2 * F, H, **kw)
        eng.moe_combine(ty, self.drows, self.pos, None, n, k, H, self.dx, p, **kw)

    def check(self):
        """Against automatic differentiation in 64 bits. Every result has gone through at most seven roundings to the rows' type (half a step
        each) and sums of in all under 1000 terms in fp32 (2^-23 each), of values that are at most some 16 times the result's
        largest."""
        import torch
        torch.cuda.synchronize()
        live, F = self.live, self.ff
        leaf = lambda t: t.double().cpu().requires_grad_()  # noqa: E731
        x, gu, down, logits = leaf(self.x[:live]), leaf(self.gu), leaf(self.down), leaf(self.logits[:live])
        idx = self.idx.cpu().long().reshape(self.n, self.k)
        assert (idx[live:] == -1).all() and torch.equal(idx[:live], self.logits[:live].double().cpu().topk(self.k).indices)
        idx = idx[:live]
        w = torch.softmax(logits.gather(1, idx), 1)
        out = 0
        for s in range(self.k):
            m = (gu[idx[:, s]] @ x.unsqueeze(-1)).squeeze(-1)
            a = m[:, :F] * torch.sigmoid(m[:, :F]) * m[:, F:]
            out = out + w[:, s:s + 1] * (down[idx[:, s]] @ a.unsqueeze(-1)).squeeze(-1)
        out.backward(self.dout[:live].double().cpu())
        bound = 16 * (7 * torch.finfo(dtype(self.ty)).eps / 2 + 1000 * 2.0 ** -23)
        for name, got, want in (("out", self.out, out.detach()), ("dx", self.dx, x.grad), ("dgu", self.dgu, gu.grad), ("ddown", self.ddown, down.grad),
                                ("dlogits", self.dlogits, logits.grad)):
            got = got.double().cpu()
            if name in ("out", "dx", "dlogits"):
                assert (got[live:] == 0).all(), name
                got = got[:live]
            assert float((got - want).abs().max()) <= bound * float(want.abs().max()), name


@pytest.mark.parametrize("ty", [le.F32, le.F16, le.BF16])
@pytest.mark.parametrize("n,hidden,ff", [(3, 64, 40), (50, 136, 72), (400, 61, 33)])
def test_training_step(engine, ty, n, hidden, ff):
    t = Train(engine, ty, n, 1, hidden, ff)
    t.fill(2)
    t.run(engine)
    t.check()


def test_training_graphs_side_by_side(engine):
    """Two captured steps with workspaces of their own on two streams at once; replays with new inputs and eager steps between."""
    import torch
    ts = [Train(engine, le.BF16, 60, 3), Train(engine, le.F32, 200, 4)]
    for t in ts:
        t.fill(5)
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
        ts[1].check()
