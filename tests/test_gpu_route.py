"""GPU parity of the expert-routing entries (le_moe_route, le_moe_sort, le_moe_permute, le_moe_combine and their gradients)
against plain forms in 64 bits, alone and run together.

Tolerances, with u = 2^-24: a routing weight is exp(l - top) / sum: the subtraction is exact to u |l - top|, which the exponential
makes a relative error of the same size, expf adds 2 u, the sum of k terms k u, the division u. Sums of n products in fp32 are off
by at most (n + 1) u times the sum of the terms' magnitudes. Rounding to 16 bits adds half a step, eps / 2 of the value."""
import numpy as np
import pytest

import lastengine_amd as le

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [le.F32, le.F16, le.BF16]


def torch_type(ty):
    import torch
    return {le.F32: torch.float32, le.F16: torch.float16, le.BF16: torch.bfloat16}[ty]


def half_step(ty):
    import torch
    return 0.0 if ty == le.F32 else torch.finfo(torch_type(ty)).eps / 2


def tiny(ty):
    import torch
    f = torch.finfo(torch_type(ty))
    return f.smallest_normal * f.eps / 2


# ---------------------------------------------------------------- router

def route_plain(l, k):
    """idx, w and the largest |l - top| of each token, in 64 bits; l: float64 tensor."""
    import torch
    v = torch.where(torch.isnan(l), -torch.inf, l)
    top, order = torch.sort(v, dim=-1, descending=True, stable=True)
    top, order = top[:, :k], order[:, :k]
    there = top > -torch.inf
    first = torch.where(there[:, :1], top[:, :1], 0.0)
    d = torch.where(there, top - first, 0.0)
    e = torch.where(there, d.exp(), 0.0)
    w = e / torch.where(there[:, :1], e.sum(-1, keepdim=True), 1.0)
    return torch.where(there, order, -1).int(), w, d.abs()


def check_route(engine, l, ty, k):
    import torch
    n, n_exp = l.shape
    idx = torch.full((n * k + 8,), 99, dtype=torch.int32, device="cuda")
    w = torch.full((n * k + 8,), 99.0, device="cuda")
    print("route", tuple(l.shape), ty, k, flush=True)
    engine.moe_route(ty, l.cuda(), n, n_exp, k, idx, w)
    torch.cuda.synchronize()
    assert (idx[n * k:] == 99).all() and (w[n * k:] == 99).all()
    gi, gw = idx[:n * k].reshape(n, k).cpu(), w[:n * k].reshape(n, k).double().cpu()
    wi, ww, d = route_plain(l.double(), k)
    assert torch.equal(gi, wi)
    # numerator and denominator both carry the exponentials' errors
    far = d.max(-1, keepdim=True).values if k else d
    assert ((gw - ww).abs() <= ww * U * (d + far + k + 8) + 2.0 ** -125).all()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("n_tok,n_exp,k", [(1, 1, 1), (1, 8, 2), (3, 7, 7), (5, 60, 6), (8, 64, 8), (9, 65, 3), (33, 128, 8), (130, 256, 8), (17, 300, 16),
                                           (65, 512, 10), (6, 1000, 16), (2, 1024, 1), (5000, 128, 8), (4099, 16, 4)])
def test_route(engine, ty, n_tok, n_exp, k):
    import torch
    g = torch.Generator().manual_seed(n_tok + n_exp)
    l = (torch.randn(n_tok, n_exp, generator=g) * 3).to(torch_type(ty))  # 16-bit logits hold many equal ones
    check_route(engine, l, ty, k)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("n_exp,k", [(8, 8), (60, 4), (128, 8), (257, 16), (1024, 5)])
def test_route_masks(engine, ty, n_exp, k):
    """Ties, experts masked by -infinity, NaN or the type's lowest value, tokens with fewer than k experts or none."""
    import torch
    low = torch.finfo(torch_type(ty)).min
    g = torch.Generator().manual_seed(n_exp)
    l = torch.randn(14, n_exp, generator=g).to(torch_type(ty))
    l[0] = -torch.inf
    l[1] = torch.nan
    l[2] = low
    l[3] = 0.0
    l[4] = -torch.inf
    l[4, n_exp - 1] = low
    l[5, ::2] = -torch.inf
    l[6, 1::2] = torch.nan
    l[7, 3:] = low
    l[8] = torch.randint(0, 2, (n_exp,), generator=g).to(l.dtype)
    l[9, 2:] = -torch.inf
    l[10, 0] = torch.nan
    l[11] = torch.where(torch.arange(n_exp) % 3 == 0, torch.tensor(-0.0), torch.tensor(0.0)).to(l.dtype)  # equal
    l[12] = -torch.finfo(torch_type(ty)).tiny
    l[13, :] = torch.finfo(torch_type(ty)).max
    check_route(engine, l, ty, k)


def route_bwd_plain(idx, w, dw, n_exp):
    import torch
    ok = (idx >= 0) & (idx < n_exp)
    w, dw = torch.where(ok, w, 0.0), torch.where(ok, dw, 0.0)
    g = w * (dw - (w * dw).sum(-1, keepdim=True))
    mag = w * (dw.abs() + (w * dw.abs()).sum(-1, keepdim=True))
    at = torch.where(ok, idx, n_exp).long()
    return [torch.zeros(len(idx), n_exp + 1, dtype=torch.float64).scatter_add_(1, at, v)[:, :n_exp] for v in (g, mag)]


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("n_tok,n_exp,k", [(1, 1, 1), (2, 8, 8), (7, 60, 6), (300, 128, 8), (33, 1024, 16), (3, 65, 1), (5000, 16, 2)])
def test_route_bwd(engine, ty, n_tok, n_exp, k):
    import torch
    g = torch.Generator().manual_seed(n_exp + k)
    l = torch.randn(n_tok, n_exp, generator=g).double()
    l[n_tok // 2, 1:] = -torch.inf  # fewer than k selected
    idx, w, _ = route_plain(l, k)
    idx[0, 0] = -7 if n_tok > 1 else idx[0, 0]
    dw = torch.randn(n_tok, k, generator=g)
    dw[w == 0] = torch.nan  # nothing is read at selections without an expert
    w = w.float()
    out = torch.full((n_tok * n_exp + 8,), 9.0, dtype=torch_type(ty), device="cuda")
    print("route_bwd", ty, n_tok, n_exp, k, flush=True)
    engine.moe_route_bwd(ty, idx.cuda(), w.cuda(), dw.cuda(), n_tok, n_exp, k, out)
    torch.cuda.synchronize()
    assert (out[n_tok * n_exp:] == 9).all()
    want, mag = route_bwd_plain(idx, w.double(), dw.double(), n_exp)
    got = out[:n_tok * n_exp].reshape(n_tok, n_exp).double().cpu()
    assert ((got - want).abs() <= half_step(ty) * want.abs() + 2 * (k + 3) * U * mag + tiny(ty)).all()


def test_route_gradient_by_differences(engine):
    """dlogits against central differences of the weights' definition in 64 bits (step 1e-6: truncation ~1e-12 of the third
    derivative, cancellation ~1e-10; the fp32 result's own rounding, 2 (k + 3) u of terms below 4, is the larger: 1e-5 in all)."""
    import torch
    n_tok, n_exp, k, h = 6, 12, 4, 1e-6
    g = torch.Generator().manual_seed(4)
    l = (torch.randn(n_tok, n_exp, generator=g) * 2).double()
    dw = torch.randn(n_tok, k, generator=g).double()
    num = torch.zeros(n_tok, n_exp, dtype=torch.float64)
    for e in range(n_exp):
        d = torch.zeros(n_tok, n_exp, dtype=torch.float64)
        d[:, e] = h
        (i0, w0, _), (i1, w1, _) = route_plain(l - d, k), route_plain(l + d, k)
        assert torch.equal(i0, i1)
        num[:, e] = ((w1 - w0) * dw).sum(-1) / (2 * h)
    idx, w = torch.empty(n_tok, k, dtype=torch.int32, device="cuda"), torch.empty(n_tok, k, device="cuda")
    dl = torch.empty(n_tok, n_exp, device="cuda")
    engine.moe_route(le.F32, l.float().cuda(), n_tok, n_exp, k, idx, w)
    engine.moe_route_bwd(le.F32, idx, w, dw.float().cuda(), n_tok, n_exp, k, dl)
    assert float((dl.double().cpu() - num).abs().max()) <= 1e-5


# ---------------------------------------------------------------- sort

def sort_plain(idx, k, n_exp):
    p = idx.reshape(-1).astype(np.int64)
    ok = (p >= 0) & (p < n_exp)
    order = np.argsort(np.where(ok, p, n_exp), kind="stable")[:int(ok.sum())]
    off = np.concatenate([[0], np.cumsum(np.bincount(p[ok], minlength=n_exp))]).astype(np.int32)
    pos = np.full(len(p), -1, np.int32)
    pos[order] = np.arange(len(order))
    return off, (order // k).astype(np.int32), order.astype(np.int32), pos


def check_sort(engine, idx, n_tok, k, n_exp, stream=None):
    import torch
    n = n_tok * k
    d = torch.from_numpy(np.ascontiguousarray(idx, dtype=np.int32)).cuda()
    off = torch.full((n_exp + 1 + 4,), 55, dtype=torch.int32, device="cuda")
    i, o, p = (torch.full((n + 4,), 55, dtype=torch.int32, device="cuda") for _ in range(3))
    nws = engine.moe_sort_workspace_size(n_tok, k, n_exp)
    ws = torch.full((nws + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    print("sort", n_tok, k, n_exp, nws, flush=True)
    engine.moe_sort(d, n_tok, k, n_exp, off, i, o, p, ws=ws, ws_bytes=nws)
    torch.cuda.synchronize()
    assert (ws[nws:] == 0xA5).all()
    w_off, w_in, w_out, w_pos = sort_plain(np.asarray(idx), k, n_exp)
    live = len(w_in)
    for got, want in ((off, w_off), (i, w_in), (o, w_out), (p, w_pos)):
        assert np.array_equal(got.cpu().numpy()[:len(want)], want)
    assert (off[n_exp + 1:] == 55).all() and (p[n:] == 55).all() and (i[live:] == 55).all() and (o[live:] == 55).all()
    return d, w_off, w_pos


SORTS = [(0, 1, 1), (0, 8, 128), (1, 1, 1), (1, 8, 128), (3, 5, 7), (8, 8, 128), (37, 8, 128), (64, 1, 64), (63, 16, 1024), (65, 4, 65), (100, 6, 60),
         (128, 8, 256), (513, 8, 128), (2049, 2, 8), (4096, 8, 128), (5000, 7, 1000), (16385, 4, 33), (65536, 8, 128), (70000, 16, 256)]


@pytest.mark.parametrize("n_tok,k,n_exp", SORTS)
@pytest.mark.parametrize("what", ["even", "one", "skewed", "dropped", "none"])
def test_sort(engine, n_tok, k, n_exp, what):
    rng = np.random.default_rng(n_tok + k + n_exp)
    n = n_tok * k
    idx = rng.integers(0, n_exp, size=n)
    if what == "one":
        idx[:] = n_exp - 1
    elif what == "skewed":
        idx = np.minimum(rng.geometric(0.3, size=n) - 1, n_exp - 1)
    elif what == "dropped":  # padding, experts of another rank, anything
        idx = np.where(rng.random(n) < 0.4, rng.choice([-1, n_exp, -2**31, 2**31 - 1, n_exp + 5], size=n), idx)
    elif what == "none":
        idx[:] = -1
    check_sort(engine, idx, n_tok, k, n_exp)


@pytest.mark.parametrize("n_tok", [5, 6000])
def test_sort_optional_outputs(engine, n_tok):
    import torch
    k, n_exp = 4, 40
    idx = np.random.default_rng(1).integers(-1, n_exp, size=n_tok * k)
    d, w_off, w_pos = check_sort(engine, idx, n_tok, k, n_exp)
    off = torch.empty(n_exp + 1, dtype=torch.int32, device="cuda")
    engine.moe_sort(d, n_tok, k, n_exp, off)
    assert np.array_equal(off.cpu().numpy(), w_off)
    pos = torch.empty(n_tok * k, dtype=torch.int32, device="cuda")
    engine.moe_sort(d, n_tok, k, n_exp, off, pos=pos)
    assert np.array_equal(pos.cpu().numpy(), w_pos)


# ---------------------------------------------------------------- rows

def positions(n_tok, k, n_row, seed, dropped=0.2):
    """Distinct rows for the pairs (as far as they go), some pairs without one, numbers outside the rows among those."""
    rng = np.random.default_rng(seed)
    n = n_tok * k
    pos = np.full(n, -1, np.int64)
    take = min(n, n_row)
    pos[rng.permutation(n)[:take]] = rng.permutation(n_row)[:take]
    drop = rng.random(n) < dropped
    pos[drop] = rng.choice([-1, n_row, -2**31, 2**31 - 1], size=int(drop.sum()))
    return pos.astype(np.int32)


class Rows:
    """n rows of cols values, ld apart, from an address `shift` values behind an aligned one; 66 between them."""

    def __init__(self, n, cols, ld, ty, shift, fill=None, seed=0):
        import torch
        self.buf = torch.full((n * ld + shift + 16,), 66.0, dtype=torch_type(ty), device="cuda")
        self.n, self.cols, self.ld, self.at = n, cols, ld, shift
        self.ptr = self.buf[shift:]
        if fill == "normal":
            self.view().copy_(torch.randn(n, cols, generator=torch.Generator().manual_seed(seed)).to(torch_type(ty)))
        self.before = self.buf.clone()

    def view(self):
        return self.buf[self.at:self.at + self.n * self.ld].reshape(self.n, self.ld)[:, :self.cols]

    def rest_is_kept(self, rows=None):
        import torch
        """Nothing but the given rows' values changed."""
        a, b = self.before.clone(), self.buf.clone()
        for v in (a, b):
            w = v[self.at:self.at + self.n * self.ld].reshape(self.n, self.ld)[:, :self.cols]
            if rows is None:
                w.zero_()
            else:
                w[rows] = 0
        return torch.equal(a, b)


ROWS = [  # n_tok, k, cols, token stride - cols, expert stride - cols, shift of both in values
    (1, 1, 1, 0, 0, 0), (1, 8, 2048, 0, 0, 0), (5, 3, 7, 0, 0, 0), (4, 2, 8, 0, 0, 1), (37, 8, 1001, 0, 0, 0), (9, 6, 1000, 24, 8, 0),
    (6, 4, 2047, 1, 3, 1), (3, 16, 5000, 0, 8, 0), (130, 4, 72, 8, 0, 2), (2, 2, 20000, 0, 0, 0), (700, 2, 64, 0, 0, 0), (300, 8, 256, 0, 0, 0),
    (4, 8, 4096, 0, 0, 4)]


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("n_tok,k,cols,dt,de,shift", ROWS)
def test_permute(engine, ty, n_tok, k, cols, dt, de, shift):
    import torch
    n_row = n_tok * k + 3
    pos = positions(n_tok, k, n_row, cols)
    x, e = Rows(n_tok, cols, cols + dt, ty, shift, "normal", 1), Rows(n_row, cols, cols + de, ty, shift)
    print("permute", ty, n_tok, k, cols, dt, de, shift, flush=True)
    engine.moe_permute(ty, x.ptr, torch.from_numpy(pos).cuda(), n_tok, k, cols, e.ptr, n_row, ldt=x.ld, lde=e.ld)
    torch.cuda.synchronize()
    live = np.flatnonzero((pos >= 0) & (pos < n_row))
    assert torch.equal(e.view()[pos[live]], x.view()[live // k])
    assert e.rest_is_kept(torch.from_numpy(pos[live]).long().cuda())


def combine_plain(rows, pos, w, n_tok, k):
    """The sum and the sum of its terms' magnitudes, in 64 bits; rows that no pair names are not looked at."""
    import torch
    rows = rows.double().cpu()
    out, mag = (torch.zeros(n_tok, rows.shape[1], dtype=torch.float64) for _ in range(2))
    for p, r in enumerate(pos):
        if 0 <= r < len(rows):
            t = rows[r] * (float(w[p]) if w is not None else 1.0)
            out[p // k] += t
            mag[p // k] += t.abs()
    return out, mag


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("weights", [True, False])
@pytest.mark.parametrize("n_tok,k,cols,dt,de,shift", ROWS)
def test_combine(engine, ty, weights, n_tok, k, cols, dt, de, shift):
    import torch
    n_row = n_tok * k + 3
    pos = positions(n_tok, k, n_row, cols + 1)
    if n_tok > 2:
        pos[k:2 * k] = -1  # a token without any
    e, out = Rows(n_row, cols, cols + de, ty, shift, "normal", 2), Rows(n_tok, cols, cols + dt, ty, shift)
    unused = np.setdiff1d(np.arange(n_row), pos)
    e.view()[unused] = float("nan")
    w = torch.randn(n_tok * k, generator=torch.Generator().manual_seed(3)) if weights else None
    if w is not None:
        w[torch.from_numpy((pos < 0) | (pos >= n_row))] = float("nan")  # not read, or read and left out
    print("combine", ty, weights, n_tok, k, cols, dt, de, shift, flush=True)
    engine.moe_combine(ty, e.ptr, torch.from_numpy(pos).cuda(), w.cuda() if weights else None, n_tok, k, cols, out.ptr, n_row, ldt=out.ld, lde=e.ld)
    torch.cuda.synchronize()
    want, mag = combine_plain(e.view(), pos, w, n_tok, k)
    err = (out.view().double().cpu() - want).abs()
    assert (err <= half_step(ty) * want.abs() + 2 * (k + 1) * U * mag + tiny(ty)).all()
    assert out.rest_is_kept()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("outputs", ["both", "rows", "weights", "in place"])
@pytest.mark.parametrize("n_tok,k,cols,dt,de,shift", ROWS)
def test_combine_bwd(engine, ty, outputs, n_tok, k, cols, dt, de, shift):
    import torch
    n_row = n_tok * k + 3
    pos = positions(n_tok, k, n_row, cols + 2)
    g, e = Rows(n_tok, cols, cols + dt, ty, shift, "normal", 4), Rows(n_row, cols, cols + de, ty, shift, "normal", 5)
    rows = e.view().double().cpu()
    d = e if outputs == "in place" else Rows(n_row, cols, cols + de, ty, shift)
    weights = cols != 2048
    w = torch.randn(n_tok * k, generator=torch.Generator().manual_seed(6)) if weights else torch.ones(n_tok * k)
    dw = torch.full((n_tok * k + 4,), 8.0, device="cuda")
    print("combine_bwd", ty, outputs, n_tok, k, cols, dt, de, shift, flush=True)
    engine.moe_combine_bwd(ty, g.ptr, e.ptr if outputs != "rows" else None, torch.from_numpy(pos).cuda(), w.cuda() if weights else None, n_tok, k, cols,
                           None if outputs == "weights" else d.ptr, None if outputs == "rows" else dw, n_row, ldt=g.ld, lde=e.ld)
    torch.cuda.synchronize()
    ok = (pos >= 0) & (pos < n_row)
    live = np.flatnonzero(ok)
    dout = g.view().double().cpu()
    if outputs != "weights":
        want = dout[live // k] * w.double()[live, None]
        got = d.view()[pos[live]].double().cpu()
        assert ((got - want).abs() <= (half_step(ty) + 2 * U) * want.abs() + tiny(ty)).all()
        assert d.rest_is_kept(torch.from_numpy(pos[live]).long().cuda())
    else:
        assert d.rest_is_kept(torch.zeros(0, dtype=torch.long).cuda())
    if outputs != "rows":
        terms = dout[live // k] * rows[pos[live]]
        got = dw[:n_tok * k].double().cpu()
        assert ((got[live] - terms.sum(1)).abs() <= (cols + 1) * U * terms.abs().sum(1) + 2.0 ** -126).all()
        assert (got[~ok] == 0).all()
    assert (dw[n_tok * k:] == 8).all()


@pytest.mark.parametrize("ty", TYPES)
def test_rows_in_pair_order(engine, ty):
    """pos None: pair p's row is row p, as far as there are rows."""
    import torch
    n_tok, k, cols, n_row = 7, 3, 40, 20  # the last pair has none
    pos = np.arange(n_tok * k).astype(np.int32)
    e = Rows(n_row, cols, cols, ty, 0, "normal", 7)
    out = Rows(n_tok, cols, cols, ty, 0)
    engine.moe_combine(ty, e.ptr, None, None, n_tok, k, cols, out.ptr, n_row)
    want, mag = combine_plain(e.view(), np.where(pos < n_row, pos, -1), None, n_tok, k)
    assert ((out.view().double().cpu() - want).abs() <= half_step(ty) * want.abs() + 2 * (k + 1) * U * mag + tiny(ty)).all()
    engine.moe_permute(ty, out.ptr, None, n_tok, k, cols, e.ptr, n_row)
    assert torch.equal(e.view(), out.view().repeat_interleave(k, 0)[:n_row]) and e.rest_is_kept()
    dw = torch.empty(n_tok * k, device="cuda")
    engine.moe_combine_bwd(ty, out.ptr, e.ptr, None, None, n_tok, k, cols, None, dw, n_row)
    assert float(dw[-1]) == 0 and float(dw[0]) > 0


def test_zero_tokens(engine):
    import torch
    t = torch.full((64,), 3.0, device="cuda")
    i = torch.full((64,), 3, dtype=torch.int32, device="cuda")
    engine.moe_route(le.F32, t, 0, 8, 2, i, t)
    engine.moe_route_bwd(le.F32, i, t, t, 0, 8, 2, t)
    engine.moe_permute(le.F32, t, i, 0, 2, 4, t, 8)
    engine.moe_combine(le.F32, t, i, t, 0, 2, 4, t, 8)
    engine.moe_combine_bwd(le.F32, t, t, i, t, 0, 2, 4, t, t, 8)
    torch.cuda.synchronize()
    assert (t == 3).all() and (i == 3).all()
    engine.moe_combine(le.F32, t, i, t, 2, 2, 4, t[32:], 0)  # no expert rows at all
    assert (t[32:40] == 0).all() and (t[:32] == 3).all() and (t[40:] == 3).all()


def test_far_rows(engine):
    """Rows whose offsets pass 32 bits, in values."""
    import torch
    cols, lde, n_row = 64, 1 << 20, 4200  # 4.4e9 bf16 values
    e = torch.empty(n_row * lde, dtype=torch.bfloat16, device="cuda")
    x = torch.randn(2, cols, device="cuda").bfloat16()
    pos = torch.tensor([0, n_row - 1, 4100, n_row], dtype=torch.int32, device="cuda")
    engine.moe_permute(le.BF16, x, pos, 2, 2, cols, e, n_row, lde=lde)
    rows = e.reshape(n_row, lde)
    assert torch.equal(rows[0, :cols], x[0]) and torch.equal(rows[n_row - 1, :cols], x[0]) and torch.equal(rows[4100, :cols], x[1])
    out = torch.empty(2, cols, dtype=torch.bfloat16, device="cuda")
    engine.moe_combine(le.BF16, e, pos, None, 2, 2, cols, out, n_row, lde=lde)
    assert torch.equal(out[0].float(), 2 * x[0].float()) and torch.equal(out[1], x[1])
    dw = torch.empty(4, device="cuda")
    engine.moe_combine_bwd(le.BF16, x, e, pos, None, 2, 2, cols, e, dw, n_row, lde=lde)
    assert torch.equal(rows[4100, :cols], x[1]) and float(dw[3]) == 0
    want = x[1].double().square().sum()
    assert abs(float(dw[2]) - float(want)) <= cols * U * float(want)


def test_refusals(engine):
    import torch
    t = torch.zeros(64, device="cuda")
    i = torch.zeros(64, dtype=torch.int32, device="cuda")
    for call, code in ((lambda: engine.moe_route(le.Q4_K, t, 2, 8, 2, i, t), -2), (lambda: engine.moe_route(le.F32, t, 2, 4, 5, i, t), -3),
                       (lambda: engine.moe_sort(i, 2, 17, 8, i), -3), (lambda: engine.moe_sort(i, 2, 2, 8, None), -1),
                       (lambda: engine.moe_permute(le.F32, t, i, 2, 2, 8, t, 4, ldt=4), -3), (lambda: engine.moe_combine(le.F32, t, i, t, 2, 2, 0, t, 4), -3),
                       (lambda: engine.moe_combine_bwd(le.F32, None, t, i, t, 2, 2, 8, t, t, 4), -1)):
        with pytest.raises(le.LeError) as e:
            call()
        assert e.value.code == code


@pytest.mark.parametrize("ty", TYPES)
def test_many_rows(engine, ty):
    """Enough aligned rows for the non-temporal loads, with the last token's pairs and some others without a row."""
    import torch
    n_tok, k, cols = 1100, 8, 1024 if ty == le.F32 else 2048
    n_row = n_tok * k
    pos = positions(n_tok, k, n_row, 5, 0.05)
    pos[-k:] = -1
    g = torch.Generator().manual_seed(8)
    e = torch.randn(n_row, cols, generator=g).to(torch_type(ty)).cuda()
    dout = torch.randn(n_tok, cols, generator=g).to(torch_type(ty)).cuda()
    w = torch.randn(n_tok * k, generator=g).cuda()
    dpos = torch.from_numpy(pos).cuda()
    out = torch.empty(n_tok, cols, dtype=torch_type(ty), device="cuda")
    de, dw = torch.zeros_like(e), torch.empty(n_tok * k, device="cuda")
    engine.moe_combine(ty, e, dpos, w, n_tok, k, cols, out, n_row)
    engine.moe_combine_bwd(ty, dout, e, dpos, w, n_tok, k, cols, de, dw, n_row)
    ok = ((dpos >= 0) & (dpos < n_row)).reshape(n_tok, k)
    at = torch.where(ok, dpos.reshape(n_tok, k), 0).long()
    ww = torch.where(ok, w.reshape(n_tok, k), 0.0).double()
    rows = e.double()[at]
    want, mag = (rows * ww[..., None]).sum(1), (rows * ww[..., None]).abs().sum(1)
    assert ((out.double() - want).abs() <= half_step(ty) * want.abs() + 2 * (k + 1) * U * mag + tiny(ty)).all() and (out[-1] == 0).all()
    terms = dout.double()[:, None] * rows
    got = dw.double().reshape(n_tok, k)
    assert ((got - terms.sum(-1)).abs() <= (cols + 1) * U * terms.abs().sum(-1))[ok].all() and (got[~ok] == 0).all()
    grad = torch.zeros_like(e, dtype=torch.float64)
    grad[at[ok]] = (dout.double()[:, None] * ww[..., None])[ok]
    assert ((de.double() - grad).abs() <= (half_step(ty) + 2 * U) * grad.abs() + tiny(ty)).all()


def test_more_tokens_than_blocks(engine):
    """Token counts past the grids' limits, where blocks take several."""
    import torch
    n = (1 << 24) + 37  # sixteen tokens a block, 2^20 blocks
    l = torch.randn(n, 3, device="cuda")
    idx, w = torch.empty(n, 2, dtype=torch.int32, device="cuda"), torch.empty(n, 2, device="cuda")
    print("route", n, flush=True)
    engine.moe_route(le.F32, l, n, 3, 2, idx, w)
    top, order = torch.sort(l, dim=-1, descending=True, stable=True)
    assert torch.equal(idx, order[:, :2].int())
    assert float((w - torch.softmax(top[:, :2].double(), -1)).abs().max()) <= 1e-5
    dl = torch.empty(n, 3, device="cuda")
    dw = torch.randn(n, 2, device="cuda")
    engine.moe_route_bwd(le.F32, idx, w, dw, n, 3, 2, dl)
    g = w.double() * (dw.double() - (w.double() * dw.double()).sum(-1, keepdim=True))
    assert float((dl.double() - torch.zeros(n, 3, dtype=torch.float64, device="cuda").scatter_(1, idx.long(), g)).abs().max()) <= 1e-5
    del l, top, order, g, dl
    n, cols = (1 << 20) + 5, 520  # a block each
    x = torch.randn(n, cols, device="cuda", dtype=torch.float32)
    pos = torch.randperm(n, device="cuda").int()
    pos[3] = -1
    e, out = torch.zeros(n, cols, device="cuda"), torch.empty(n, cols, device="cuda")
    print("rows", n, flush=True)
    engine.moe_permute(le.F32, x, pos, n, 1, cols, e, n)
    engine.moe_combine(le.F32, e, pos, None, n, 1, cols, out, n)
    want = x.clone()
    want[3] = 0
    assert torch.equal(out, want)
    w = torch.randn(n, device="cuda")
    dw, de = torch.empty(n, device="cuda"), torch.zeros_like(e)
    engine.moe_combine_bwd(le.F32, x, e, pos, w, n, 1, cols, de, dw, n)
    sq = x.double().square().sum(1)
    sq[3] = 0
    assert ((dw.double() - sq).abs() <= (cols + 1) * U * sq).all()
    engine.moe_combine(le.F32, de, pos, None, n, 1, cols, out, n)
    assert ((out - want * w[:, None]).abs() <= 2 * U * (want * w[:, None]).abs() + 2.0 ** -126).all()
