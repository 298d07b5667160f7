"""GPU parity of the matrix-vector products with 4-bit codes and group scales (le_matvec_g4) against a plain form in 64 bits.

Tolerance: with u = 2^-24, the kernels add products that are exact in fp32 up to a final rounding, in some order. Codes enter
as 16 + code, the zero points through the group's sum of activations, so an output's terms are
T = sum over c of |scale| (31 + 16 + |zero|) |a|, and any order of n additions is off by at most n u T: 16 (chains of a
wave) + 2 log2... at most `cols` of them. That bound holds for every output. It is wide, so the outputs together are held to
what rounding errors of random sign add up to: an rms error of u sqrt(cols / 2) times the rms of partial sums of T's kind,
which are at most 6 times the result's where codes and activations are spread as here ((16 + code) against (code - zero),
rms 24 against 4). Rounding to 16 bits adds half a step, eps / 2 of the value (and half of the smallest subnormal)."""
import numpy as np
import pytest

import lastengine_amd as le

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def torch_type(ty):
    import torch
    return {le.F32: torch.float32, le.F16: torch.float16, le.BF16: torch.bfloat16}[ty]


def make(n_mat, rows, cols, group, stype, zeros, seed, frac=False):
    import torch
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (n_mat, rows, cols // 2), generator=g, dtype=torch.uint8)
    scales = (torch.randn(n_mat, rows, cols // group, generator=g) * 0.02).to(torch_type(stype))
    z = None
    if zeros:
        z = torch.randint(0, 16, scales.shape, generator=g).float()
        z = (z + (torch.rand(scales.shape, generator=g) if frac else 0.0)).to(torch_type(stype))
    return codes, scales, z


def dequant(codes, scales, z, group):
    """float64 weights (n_mat, rows, cols), and 47 + |zero| times |scale| at each."""
    import torch
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    s = scales.double().repeat_interleave(group, -1)
    zz = z.double().repeat_interleave(group, -1) if z is not None else torch.full_like(q, 8.0)
    return (q - zz) * s, (47 + zz.abs()) * s.abs()


def activations(x, cols, swiglu):
    x = x.double()
    return x[..., :cols] / (1 + (-x[..., :cols]).exp()) * x[..., cols:] if swiglu else x


def check(out, want, terms, ty, cols, rms=True):
    import torch
    out, eps = out.double().cpu(), torch.finfo(torch_type(ty)).eps
    assert torch.isfinite(out).all()
    half = 0.0 if ty == le.F32 else eps / 2
    tiny = torch.finfo(torch_type(ty)).smallest_normal * eps / 2
    err = (out - want).abs()
    # fp32 outputs: the bound on the sums covers the last addition's rounding
    bound = half * want.abs() + (1 + half) * (cols + 8) * U * terms + tiny + 2.0 ** -126
    assert (err <= bound).all(), float((err / bound).max())
    if rms and want.numel() >= 16:
        rel = float(err.norm() / want.norm())
        assert rel <= half + U * (1 + 6 * np.sqrt(cols / 2)), rel


def run(engine, ty, stype, n_mat, rows, cols, group, m, slots, share, sel, zeros, swiglu, seed, stride=None, x=None, frac=False, rms=True):
    import torch
    codes, scales, z = make(n_mat, rows, cols, group, stype, zeros, seed, frac)
    width = cols * (2 if swiglu else 1)
    nx = -(-slots // share) * m
    if x is None:
        x = torch.randn(nx, width, generator=torch.Generator().manual_seed(seed + 1)).to(torch_type(ty))
    buf = torch.full((nx, stride or width), float("nan"), dtype=torch_type(ty))
    buf[:, :width] = x
    w = le.G4(codes.cuda(), scales.cuda(), z.cuda() if z is not None else None, rows, cols, group, n_mat=n_mat)
    n = slots * m * rows
    out = torch.full((n + 64,), 77.0, dtype=torch_type(ty), device="cuda")
    dsel = torch.tensor(sel, dtype=torch.int32).cuda() if sel is not None else None
    print("g4", ty, stype, n_mat, rows, cols, group, m, slots, share, sel, zeros, swiglu, seed, flush=True)
    engine.mv_g4(ty, w, buf.cuda(), out, m=m, slots=slots, share=share, sel=dsel, xstride=stride, swiglu=swiglu)
    torch.cuda.synchronize()
    assert (out[n:] == 77.0).all(), "written behind the last output"
    got = out[:n].reshape(slots, m, rows)
    wf, mag = dequant(codes, scales, z, group)
    a = activations(x, cols, swiglu).reshape(-1, m, cols)
    for s in range(slots):
        mat = s if sel is None else sel[s]
        if not 0 <= mat < n_mat:
            assert (got[s] == 0).all()
            continue
        as_ = a[s // share]
        check(got[s], as_ @ wf[mat].t(), as_.abs() @ mag[mat].t(), ty, cols, rms)


TYPES = [le.F32, le.F16, le.BF16]


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("rows,cols,group", [(1, 32, 32), (15, 64, 64), (16, 96, 32), (17, 160, 160), (33, 352, 32), (50, 448, 64), (100, 512, 128),
                                             (64, 544, 544), (40, 2048, 32), (70, 2080, 32), (35, 4096, 128), (24, 5120, 1024), (18, 8192, 64),
                                             (257, 1024, 256), (31, 14336, 128), (19, 28672, 64)])
def test_sizes(engine, ty, rows, cols, group):
    run(engine, ty, le.F16, 1, rows, cols, group, 1, 1, 1, None, rows % 2 == 0, False, rows)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33, 64])
@pytest.mark.parametrize("cols,group", [(416, 32), (1152, 64), (2304, 256)])
def test_tokens(engine, ty, m, cols, group):
    run(engine, ty, le.F16, 1, 50, cols, group, m, 1, 1, None, m % 2 == 1, False, 100 + m)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 6, 8, 9, 17])
@pytest.mark.parametrize("cols,group", [(4608, 32), (5120, 64), (6272, 128), (8224, 32), (12352, 64), (16512, 128)])
def test_long_rows(engine, ty, m, cols, group):
    """Rows that one block's waves hold, in one go or several, and rows that several blocks share."""
    run(engine, ty, le.BF16, 1, 37, cols, group, m, 1, 1, None, m % 2 == 0, m == 3, 150 + m)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("stype", TYPES)
@pytest.mark.parametrize("zeros,swiglu", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("m", [1, 6])
def test_types(engine, ty, stype, zeros, swiglu, m):
    run(engine, ty, stype, 2, 37, 832, 64, m, 2, 1, None, zeros, swiglu, 200 + ty + stype)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("m", [1, 2, 4, 5, 16, 20])
@pytest.mark.parametrize("cols,group", [(96, 32), (4352, 128), (14336, 64)])
def test_swiglu(engine, ty, m, cols, group):
    run(engine, ty, le.F16, 1, 34, cols, group, m, 1, 1, None, True, True, 300 + m)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("m", [1, 3])
@pytest.mark.parametrize("share", [1, 2, 3, 8])
def test_slots(engine, ty, m, share):
    """Slots pick matrices of a stack: repeated ones, and numbers outside it."""
    run(engine, ty, le.F16, 5, 45, 480, 32, m, 8, share, [4, 0, 0, -1, 2, 5, 2**31 - 1, 3], True, False, 400 + share)
    run(engine, ty, le.BF16, 3, 20, 256, 256, m, 3, share, None, False, False, 410 + share)


def test_many_slots(engine):
    """More slots than a grid's blocks at once, each of a small matrix."""
    sel = [int(v) for v in np.random.default_rng(3).integers(-1, 7, size=3000)]
    run(engine, le.F32, le.F16, 6, 16, 64, 64, 1, 3000, 6, sel, True, False, 420)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("swiglu", [False, True])
def test_strides(engine, ty, swiglu):
    """Rows of x further apart than they are long (NaN between them), and one row for all."""
    import torch
    cols = 288
    run(engine, ty, le.F16, 3, 30, cols, 32, 2, 3, 1, None, True, swiglu, 500, stride=cols * (2 if swiglu else 1) + 24)
    codes, scales, z = make(1, 30, cols, 32, le.F16, True, 501)
    w = le.G4(codes.cuda(), scales.cuda(), z.cuda(), 30, cols, 32)
    x = torch.randn(cols * (2 if swiglu else 1)).to(torch_type(ty)).cuda()
    out = torch.empty(4, 30, dtype=torch_type(ty), device="cuda")
    engine.mv_g4(ty, w, x, out, m=4, xstride=0, swiglu=swiglu)
    one = torch.empty(30, dtype=torch_type(ty), device="cuda")
    engine.mv_g4(ty, w, x, one, m=1, swiglu=swiglu)
    got = out.double().cpu()
    want = activations(x.cpu(), cols, swiglu) @ dequant(codes, scales, z, 32)[0][0].t()
    mag = activations(x.cpu(), cols, swiglu).abs() @ dequant(codes, scales, z, 32)[1][0].t()
    for t in range(4):
        check(got[t], want, mag, ty, cols)
    check(one, want, mag, ty, cols)


@pytest.mark.parametrize("ty", TYPES)
def test_least_alignment(engine, ty):
    """scales, zeros and the output aligned to their values only."""
    import torch
    rows, cols, group = 21, 640, 64
    codes, scales, z = make(1, rows, cols, group, le.F16, True, 510)
    ds, dz = torch.zeros(scales.numel() + 1, dtype=torch.float16).cuda(), torch.zeros(z.numel() + 1, dtype=torch.float16).cuda()
    ds[1:], dz[1:] = scales.flatten().cuda(), z.flatten().cuda()
    w = le.G4(codes.cuda(), ds[1:], dz[1:], rows, cols, group)
    x = torch.randn(3, cols).to(torch_type(ty))
    out = torch.full((3 * rows + 1,), 5.0, dtype=torch_type(ty), device="cuda")
    engine.mv_g4(ty, w, x.cuda(), out[1:], m=3)
    wf, mag = dequant(codes, scales, z, group)
    check(out[1:].reshape(3, rows), x.double() @ wf[0].t(), x.double().abs() @ mag[0].t(), ty, cols)
    assert float(out[0]) == 5.0


@pytest.mark.parametrize("ty,big", [(le.F32, 1e30), (le.F32, 1e-30), (le.BF16, 1e30), (le.BF16, 1e-30), (le.F16, 1e3), (le.F16, 1e-4)])
def test_magnitudes(engine, ty, big):
    """Tokens of very different magnitudes in one call; zero points that are no whole numbers, scales of either sign."""
    import torch
    x = torch.randn(6, 1056, generator=torch.Generator().manual_seed(5))
    x[::2] *= big
    x[3] = 0
    run(engine, ty, le.F16, 1, 40, 1056, 32, 6, 1, 1, None, True, False, 520, x=x.to(torch_type(ty)), frac=True, rms=False)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("m", [2, 5, 12])
def test_not_finite(engine, ty, bad, m):
    """A token with an activation that is not finite gives nothing finite, and the others what they give without it."""
    import torch
    rows, cols = 40, 736
    codes, scales, z = make(1, rows, cols, 32, le.F16, True, 530)
    w = le.G4(codes.cuda(), scales.cuda(), z.cuda(), rows, cols, 32)
    x = torch.randn(m, cols).to(torch_type(ty))
    out, ref = (torch.empty(m, rows, dtype=torch_type(ty), device="cuda") for _ in range(2))
    engine.mv_g4(ty, w, x.cuda(), ref, m=m)
    x[1, 77] = bad
    engine.mv_g4(ty, w, x.cuda(), out, m=m)
    assert not torch.isfinite(out[1]).any()
    keep = [t for t in range(m) if t != 1]
    assert torch.equal(out[keep], ref[keep])


@pytest.mark.parametrize("ty", [le.F32, le.BF16])
@pytest.mark.parametrize("m", [1, 3, 20])
def test_far_gates(engine, ty, m):
    """Gates whose exponential, or whose product with log2 e, no fp32 holds, next to ordinary ones: SwiGLU is gate * up, or 0.

    The ups are at 2^-118 so that the products stay in range; the ordinary gates' products are below the tolerance then, and
    normal (|g| > 2^-8 nearly always, and what is flushed otherwise is 2^-126 of 1024 columns, below the bound's U * terms)."""
    import torch
    gen = torch.Generator().manual_seed(540)
    gates = torch.tensor([3e38, -3e38, 1e37, -1e37, -1000.0, 2.5e38, -88.5, -2e30])
    g = gates[torch.randint(0, 8, (m, 1024), generator=gen)]
    g[:, ::3] = torch.randn(m, 342, generator=gen)
    x = torch.cat([g, torch.randn(m, 1024, generator=gen) * 2.0 ** -118], 1).to(torch_type(ty))
    run(engine, ty, le.F16, 1, 40, 1024, 64, m, 1, 1, None, True, True, 541, x=x, rms=False)


@pytest.mark.parametrize("ty", TYPES)
def test_gates_that_are_not_finite(engine, ty):
    import torch
    codes, scales, z = make(1, 32, 512, 64, le.F16, True, 545)
    w = le.G4(codes.cuda(), scales.cuda(), z.cuda(), 32, 512, 64)
    for m in (1, 3):
        for bad in (float("inf"), float("-inf"), float("nan")):
            x = torch.randn(m, 1024).to(torch_type(ty))
            x[0, 100] = bad
            out = torch.zeros(m, 32, dtype=torch_type(ty), device="cuda")
            engine.mv_g4(ty, w, x.cuda(), out, m=m, swiglu=True)
            assert not torch.isfinite(out[0]).any() and torch.isfinite(out[1:]).all()


def test_same_bits_again(engine):
    """Sums in a fixed order: the same bits from call to call, and in a batch of another size class or not."""
    import torch
    rows, cols = 300, 4096
    codes, scales, z = make(1, rows, cols, 128, le.F16, True, 540)
    w = le.G4(codes.cuda(), scales.cuda(), z.cuda(), rows, cols, 128)
    x = torch.randn(1, cols).cuda()
    outs = [torch.empty(1, rows, device="cuda") for _ in range(5)]
    for o in outs:
        engine.mv_g4(le.F32, w, x, o)
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_far_matrix(engine):
    """A stack of more than 4 GiB of codes: offsets past 32 bits (of bytes, and of values)."""
    import torch
    rows, cols, n_mat = 4096, 16384, 140  # 4.7 GB of codes, 9.4e9 values
    codes = torch.randint(0, 256, (n_mat, rows, cols // 2), device="cuda", dtype=torch.uint8)
    scales = torch.full((n_mat, rows, 1), 0.01, dtype=torch.float16, device="cuda")
    w = le.G4(codes, scales, None, rows, cols, cols, n_mat=n_mat)
    x = torch.randn(2, cols, device="cuda")
    out = torch.empty(2, rows, device="cuda")
    sel = torch.tensor([n_mat - 1, 66], dtype=torch.int32, device="cuda")
    engine.mv_g4(le.F32, w, x, out, slots=2, sel=sel)
    for s, mat in enumerate((n_mat - 1, 66)):
        at = [0, 1, 2047, rows - 1]
        wf, mag = dequant(codes[mat:mat + 1, at].cpu(), scales[mat:mat + 1, at].cpu(), None, cols)
        a = x[s].double().cpu()
        check(out[s][at], a @ wf[0].t(), a.abs() @ mag[0].t(), le.F32, cols, rms=False)


def test_refusals(engine):
    import torch
    codes, scales, z = make(1, 16, 64, 32, le.F16, True, 550)
    w = le.G4(codes.cuda(), scales.cuda(), z.cuda(), 16, 64, 32)
    x, out = torch.zeros(2, 64, device="cuda"), torch.zeros(2, 16, device="cuda")
    for kw, code in ((dict(m=65), -3), (dict(slots=2), -3), (dict(xstride=32), -3), (dict(m=0), -3)):
        with pytest.raises(le.LeError) as e:
            engine.mv_g4(le.F32, w, x, out, **kw)
        assert e.value.code == code
    with pytest.raises(le.LeError) as e:
        engine.mv_g4(le.Q4_K, w, x, out)
    assert e.value.code == -2
    with pytest.raises(le.LeError) as e:
        engine.mv_g4(le.F32, w, x.flatten()[1:], out)
    assert e.value.code == -4
    for bad in ((codes[..., :16], scales, z, 16, 64, 32), (codes, scales, z.float(), 16, 64, 32), (codes, scales[:, :, :1], z, 16, 64, 32),
                (codes, scales.double(), None, 16, 64, 32), (codes.transpose(1, 2), scales, z, 16, 64, 32)):
        with pytest.raises(le.LeError):
            le.G4(*bad)


@pytest.mark.parametrize("ty,m,cols", [(le.F32, 5, 9216), (le.BF16, 20, 640), (le.F16, 3, 4352)])
def test_streams_and_workspaces(engine, ty, m, cols):
    """On streams given as torch streams and as raw handles, with a workspace of the call's own or the caller's, all at once."""
    import torch
    rows, group = 200, 64
    codes, scales, z = make(1, rows, cols, group, le.F16, True, 560)
    w = le.G4(codes.cuda(), scales.cuda(), z.cuda(), rows, cols, group)
    wf, mag = dequant(codes, scales, z, group)
    xs = [torch.randn(m, cols, generator=torch.Generator().manual_seed(i)).to(torch_type(ty)) for i in range(4)]
    dx = [x.cuda() for x in xs]
    outs = [torch.full((m, rows), float("nan"), dtype=torch_type(ty), device="cuda") for _ in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    need = engine.mv_g4_workspace_size(ty, w, m)
    assert need > 0
    for i, s in enumerate(streams):
        ws = torch.empty(need, dtype=torch.uint8, device="cuda") if i == 3 else None
        if ws is not None:
            ws.record_stream(s)
        engine.mv_g4(ty, w, dx[i], outs[i], m=m, ws=ws, stream=s if i != 1 else s.cuda_stream)
    engine.mv_g4(ty, w, dx[0], outs[2], m=m, stream=streams[2])  # behind the first on its stream
    torch.cuda.synchronize()
    for i, x in enumerate(xs):
        a = xs[0].double() if i == 2 else x.double()
        check(outs[i], a @ wf[0].t(), a.abs() @ mag[0].t(), ty, cols)
    with pytest.raises(le.LeError) as e:
        engine.mv_g4(ty, w, dx[0], outs[0], m=m, ws=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
    assert e.value.code == -7


def test_workspace_of_another_stream(engine):
    """A call on another stream takes no memory that the current stream's work may still use."""
    import torch
    from lastengine_amd import qmm
    s = torch.cuda.Stream()
    for stream in (s, s.cuda_stream):
        used = torch.empty(37 << 20, dtype=torch.uint8, device="cuda")
        at = used.data_ptr()
        del used  # free for the current stream at once, for others when its work is done
        assert qmm._workspace(37 << 20, stream).data_ptr() != at
    assert qmm._workspace(37 << 20, None).data_ptr() == at and qmm._workspace(0, s) is None


@pytest.mark.parametrize("ty,m", [(le.F32, 1), (le.F32, 6), (le.BF16, 33)])
def test_graph(engine, ty, m):
    """Captured and replayed with new activations and selections, eager calls between."""
    import torch
    from tests.test_gpu_graphs import capture
    n_mat, rows, cols, group = 3, 90, 4736, 128
    codes, scales, z = make(n_mat, rows, cols, group, le.F16, True, 570)
    w = le.G4(codes.cuda(), scales.cuda(), z.cuda(), rows, cols, group, n_mat=n_mat)
    wf, mag = dequant(codes, scales, z, group)
    x = torch.zeros(m, cols, dtype=torch_type(ty), device="cuda")
    sel = torch.zeros(2, dtype=torch.int32, device="cuda")
    out = torch.zeros(2, m, rows, dtype=torch_type(ty), device="cuda")
    ws = torch.empty(max(16, engine.mv_g4_workspace_size(ty, w, m, 2, 2)), dtype=torch.uint8, device="cuda")
    call = lambda s: engine.mv_g4(ty, w, x, out, m=m, slots=2, share=2, sel=sel, ws=ws, stream=s)  # noqa: E731
    graph = capture(call)
    for rep in range(4):
        h = torch.randn(m, cols, generator=torch.Generator().manual_seed(rep)).to(torch_type(ty))
        x.copy_(h)
        sel.copy_(torch.tensor([rep % 3, (rep + 2) % 3 if rep else -1], dtype=torch.int32))
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        call(None)
        torch.cuda.synchronize()
        assert torch.equal(got, out)
        for s, mat in enumerate(sel.tolist()):
            if mat < 0:
                assert (got[s] == 0).all()
            else:
                check(got[s], h.double() @ wf[mat].t(), h.double().abs() @ mag[mat].t(), ty, cols)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("m", [1, 3, 9])
def test_scales_that_are_not_finite(engine, ty, m):
    """An infinite or NaN scale or zero point reaches its own row alone."""
    import torch
    rows, cols, group = 40, 320, 32
    codes, scales, z = make(1, rows, cols, group, le.F16, True, 580)
    clean = le.G4(codes.cuda(), scales.cuda(), z.cuda(), rows, cols, group)
    s2, z2 = scales.clone(), z.clone()
    s2[0, 7, 3], s2[0, 39, 9], z2[0, 16, 0] = float("inf"), float("nan"), float("-inf")
    x = torch.randn(m, cols).to(torch_type(ty)).cuda()
    a, b = (torch.empty(m, rows, dtype=torch_type(ty), device="cuda") for _ in range(2))
    engine.mv_g4(ty, clean, x, a, m=m)
    engine.mv_g4(ty, le.G4(codes.cuda(), s2.cuda(), z2.cuda(), rows, cols, group), x, b, m=m)
    keep = [r for r in range(rows) if r not in (7, 16, 39)]
    assert torch.equal(a[:, keep], b[:, keep]) and not torch.isfinite(b[:, [7, 16, 39]]).any()
