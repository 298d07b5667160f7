"""Argument checks and launches of le_mm_experts and its gradients, le_lora and le_add_rms_quant, without a GPU: their host sources are
compiled against a context whose launches are only written down."""
import ctypes
import os
import shutil
import subprocess

import pytest

from lastengine_amd import build, qmm
from tests.conftest import REPO
from tests.test_g4_route_args import STUB, A, Ctx

PARTS = ("ex0", "ex1", "ex30", "lo0", "lo1", "lo30", "nq")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if not shutil.which("g++") or not os.path.exists(os.path.join(build.ROCM, "include", "hip", "hip_runtime.h")):
        pytest.skip("no g++ or HIP headers")
    d = tmp_path_factory.mktemp("args")
    (d / "stub.cpp").write_text(STUB)
    so = str(d / "libargs.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I" + build.ROCM + "/include", "-I" + build.CSRC,
                    "-I" + os.path.join(REPO, "include"), str(d / "stub.cpp")] + [os.path.join(build.CSRC, f) for f in ("le_experts.cpp", "le_lora.cpp", "le_norm.cpp")] +
                   ["-o", so], check=True)
    L, real = ctypes.CDLL(so), qmm.lib()
    for name in ("le_mm_experts", "le_mm_experts_dx", "le_mm_experts_dw", "le_mm_experts_dw_workspace_size", "le_lora", "le_lora_workspace_size",
                 "le_add_rms_quant"):
        getattr(L, name).restype, getattr(L, name).argtypes = getattr(real, name).restype, getattr(real, name).argtypes
    return L


@pytest.fixture
def ctx():
    return Ctx()


class Calls:
    """Each entry with arguments that it takes, any of which can be replaced."""

    def __init__(self, lib, ctx):
        self.lib, self.ctx = lib, ctypes.addressof(ctx) if ctx is not None else None

    def y(self, ty=0, w=A, off=A, n_exp=4, x=A, ldx=64, y=A, ldy=32, n_row=100, rows=32, cols=64):
        return self.lib.le_mm_experts(self.ctx, ty, w, off, n_exp, x, ldx, y, ldy, n_row, rows, cols, None)

    def dx(self, ty=0, w=A, off=A, n_exp=4, x=A, ldx=64, y=A, ldy=32, n_row=100, rows=32, cols=64):
        return self.lib.le_mm_experts_dx(self.ctx, ty, w, off, n_exp, y, ldy, x, ldx, n_row, rows, cols, None)

    def dw(self, ty=0, w=A, off=A, n_exp=4, x=A, ldx=64, y=A, ldy=32, n_row=100, rows=32, cols=64, dwtype=None, ws=A, ws_bytes=1 << 50):
        return self.lib.le_mm_experts_dw(self.ctx, ty, y, ldy, x, ldx, off, n_exp, ty if dwtype is None else dwtype, w, n_row, rows, cols, ws, ws_bytes, None)

    def lora(self, a=A, b=A, scale=A, n_ad=3, rank=16, rows=32, cols=64, ltype=1, idx=A, xtype=0, x=A, ldx=64, m=5, base=A, ldb=32, y=A, ldy=32, ws=A,
             ws_bytes=1 << 50, ad=True):
        s = qmm._Adapters(a, b, scale, n_ad, rank, rows, cols, ltype)
        return self.lib.le_lora(self.ctx, ctypes.addressof(s) if ad else None, idx, xtype, x, ldx, m, base, ldb, y, ldy, ws, ws_bytes, None)

    def norm(self, ty=0, x=A, ldx=64, res=A, ldr=64, w=A, h=2 * A, ldh=64, o=A, ldo=64, xq=A, xd=A, xs=A, m=5, n=64, eps=1e-5):
        return self.lib.le_add_rms_quant(self.ctx, ty, x, ldx, res, ldr, w, h, ldh, o, ldo, xq, xd, xs, m, n, eps, None)


@pytest.fixture
def call(lib, ctx):
    return Calls(lib, ctx)


def fine(ctx):
    for name, g, block, lds in ctx.calls():
        assert g[0] * block < 2**32 and g[1] <= 65535 and g[2] <= 65535 and min(g) > 0 and block <= 1024 and lds <= 160 * 1024, (name, g, block, lds)


@pytest.mark.parametrize("what", ["y", "dx", "dw"])
@pytest.mark.parametrize("bad,code", [
    (dict(ty=12), -2), (dict(ty=-1), -2), (dict(n_exp=0), -3), (dict(n_exp=1025), -3), (dict(n_exp=-1), -3), (dict(n_row=-1), -3), (dict(n_row=2**30 + 1), -3),
    (dict(rows=0), -3), (dict(cols=0), -3), (dict(rows=-4), -3), (dict(rows=2**24 + 1, ldy=2**25), -3), (dict(cols=2**24 + 1, ldx=2**25), -3),
    (dict(ldx=63), -3), (dict(ldy=31), -3), (dict(ldx=-64), -3), (dict(ldx=0), -3), (dict(w=None), -1), (dict(off=None), -1), (dict(x=None), -1), (dict(y=None), -1),
    (dict(w=A + 2), -4), (dict(x=A + 2), -4), (dict(y=A + 1), -4), (dict(off=A + 2), -4), (dict(ty=1, w=A + 1), -4), (dict(ty=30, x=A + 1), -4)])
def test_experts_refusals(call, ctx, what, bad, code):
    assert getattr(call, what)(**bad) == code
    assert ctx.launches == 0 and ctx.err


@pytest.mark.parametrize("bad,code", [(dict(ty=1, dwtype=30), -2), (dict(dwtype=1), -2), (dict(ty=30, dwtype=8), -2), (dict(ws=A + 8), -4), (dict(ty=1, dwtype=0, w=A + 2), -4),
                                      (dict(n_exp=1024, rows=2**20, cols=2**20, ldx=2**20, ldy=2**20), -3)])
def test_dw_refusals(call, ctx, bad, code):
    assert call.dw(**bad) == code
    assert ctx.launches == 0 and ctx.err


def test_dw_workspace(lib, call):
    """What is asked for is taken, one byte less refused, at any size; sizes that the entry refuses need none."""
    for ty in (0, 1, 30):
        for n_exp, n_row, rows, cols in ((1, 100000, 64, 64), (1, 5, 2048, 2048), (4, 4096, 256, 256), (128, 32768, 1536, 2048), (2, 0, 8, 8)):
            n = lib.le_mm_experts_dw_workspace_size(ty, n_exp, n_row, rows, cols)
            kw = dict(ty=ty, n_exp=n_exp, n_row=n_row, rows=rows, cols=cols, ldx=cols, ldy=rows)
            assert call.dw(ws_bytes=n, **kw) == 0
            if n:
                assert call.dw(ws_bytes=n - 1, **kw) == -7 and call.dw(ws=None, **kw) == -7
            else:
                assert call.dw(ws=None, ws_bytes=0, **kw) == 0
    for bad in ((12, 1, 100000, 64, 64), (0, 0, 100000, 64, 64), (0, 1, -1, 64, 64), (0, 1, 100000, 0, 64), (0, 1, 100000, 64, -1)):
        assert lib.le_mm_experts_dw_workspace_size(*bad) == 0


@pytest.mark.parametrize("good", [
    dict(), dict(ldx=100, ldy=33), dict(n_row=1), dict(n_row=2**30), dict(n_exp=1024), dict(rows=1, cols=1), dict(rows=2**24, ldy=2**24, n_row=1),
    dict(cols=2**24, ldx=2**24, n_row=3), dict(rows=2**17, cols=2**17, ldx=2**17, ldy=2**17, n_row=2**17, n_exp=8), dict(ty=1, w=A + 2, x=A + 2, y=A + 2), dict(ty=30)])
def test_experts_launches(call, ctx, good):
    for what in ("y", "dx", "dw"):
        assert getattr(call, what)(**good) == 0, ctx.err
        fine(ctx)
    assert ctx.launches >= 3


def test_without_rows(call, ctx):
    """Nothing to do for y and dx; the weights' gradient is zeros, which a launch writes."""
    assert call.y(n_row=0, x=None, y=None) == 0 and call.dx(n_row=0, x=None, y=None) == 0 and ctx.launches == 0
    assert call.dw(n_row=0, x=None, y=None) == 0 and ctx.launches >= 1


@pytest.mark.parametrize("bad,code", [
    (dict(ad=False), -1), (dict(xtype=8), -2), (dict(ltype=12), -2), (dict(n_ad=0), -3), (dict(rank=0), -3), (dict(rank=257), -3), (dict(rows=0), -3), (dict(cols=-1), -3),
    (dict(rows=2**24 + 1, ldb=2**25, ldy=2**25), -3), (dict(cols=2**24 + 1, ldx=2**25), -3), (dict(m=-1), -3), (dict(m=1048561), -3), (dict(ldx=63), -3),
    (dict(ldx=-64), -3), (dict(ldb=31), -3), (dict(ldy=31), -3), (dict(a=None), -1), (dict(b=None), -1), (dict(idx=None), -1), (dict(x=None), -1), (dict(y=None), -1),
    (dict(a=A + 1), -4), (dict(b=A + 1), -4), (dict(ltype=0, a=A + 2), -4), (dict(scale=A + 2), -4), (dict(idx=A + 1), -4), (dict(x=A + 2), -4), (dict(base=A + 2), -4),
    (dict(y=A + 2), -4), (dict(ws=A + 8), -4), (dict(ws=None), -7), (dict(ws_bytes=5 * 16 * 4 - 1), -7), (dict(base=A, y=A, ldb=40), -1)])
def test_lora_refusals(call, ctx, bad, code):
    assert call.lora(**bad) == code
    assert ctx.launches == 0 and ctx.err


@pytest.mark.parametrize("good", [
    dict(), dict(base=None, ldb=0), dict(scale=None), dict(ldx=0), dict(rank=1), dict(rank=256), dict(m=1), dict(m=1048560), dict(rows=1, cols=1), dict(y=2 * A, ldy=50),
    dict(rows=2**24, ldb=2**24, ldy=2**24), dict(cols=2**24, ldx=2**24), dict(n_ad=100000), dict(xtype=30, ltype=30, x=A + 2, a=A + 2, b=A + 2)])
def test_lora_launches(call, ctx, good):
    assert call.lora(**good) == 0, ctx.err
    assert 1 <= ctx.launches <= 4
    fine(ctx)


def test_lora_workspace(lib, call, ctx):
    def size(xtype, m, n_ad=3, rank=16, rows=32, cols=64, ltype=1):
        s = qmm._Adapters(A, A, A, n_ad, rank, rows, cols, ltype)
        return lib.le_lora_workspace_size(ctypes.addressof(s), xtype, m)

    for m in (1, 5, 64, 4096):
        for kw in (dict(), dict(rank=256, cols=14336), dict(rank=7, cols=4096), dict(ltype=0)):
            n = size(0, m, **kw)
            assert n >= m * kw.get("rank", 16) * 4
            ldx = kw.get("cols", 64)
            assert call.lora(m=m, ws_bytes=n, ldx=ldx, **kw) == 0 and call.lora(m=m, ws_bytes=n - 1, ldx=ldx, **kw) == -7
    assert size(8, 5) == 0 and size(0, -1) == 0 and size(0, 5, rank=0) == 0 and size(0, 5, ltype=12) == 0 and size(0, 0) == 0
    assert lib.le_lora_workspace_size(None, 0, 5) == 0
    ctx.launches = 0
    assert call.lora(m=0, idx=None, x=None, y=None, ws=None, ws_bytes=0) == 0 and ctx.launches == 0


@pytest.mark.parametrize("bad,code", [
    (dict(ty=8), -2), (dict(m=-1), -3), (dict(n=0), -3), (dict(n=2**24 + 32), -3), (dict(n=40), -3), (dict(ldx=63), -3), (dict(ldr=63), -3), (dict(ldh=63), -3), (dict(ldo=63), -3),
    (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(eps=float("inf")), -1), (dict(xq=None), -1), (dict(xd=None), -1), (dict(xq=None, xd=None), -1),
    (dict(x=None), -1), (dict(w=None), -1), (dict(h=None, o=None, xq=None, xd=None, xs=None), -1), (dict(x=3 * A, h=3 * A, ldh=65), -1), (dict(res=3 * A, h=3 * A, ldh=65), -1),
    (dict(x=A + 2), -4), (dict(res=A + 2), -4), (dict(h=A + 2), -4), (dict(o=A + 1), -4), (dict(w=A + 2), -4), (dict(xd=A + 2), -4), (dict(xs=A + 1), -4), (dict(ty=1, x=A + 1), -4)])
def test_norm_refusals(call, ctx, bad, code):
    assert call.norm(**bad) == code
    assert ctx.launches == 0 and ctx.err


@pytest.mark.parametrize("good", [
    dict(), dict(res=None, ldr=0), dict(h=None, ldh=0), dict(o=None, ldo=0), dict(xs=None), dict(xq=None, xd=None, xs=None, n=63), dict(x=3 * A, h=3 * A), dict(res=3 * A, h=3 * A),
    dict(m=2**31 - 1), dict(n=2**24, ldx=2**24, ldr=2**24, ldh=2**24, ldo=2**24), dict(n=32), dict(eps=0.0), dict(ty=30, x=A + 2, res=A + 2, h=A + 4, o=A + 2), dict(xq=A + 1)])
def test_norm_launches(call, ctx, good):
    assert call.norm(**good) == 0, ctx.err
    assert ctx.launches == 1
    fine(ctx)


def test_norm_without_rows(call, ctx):
    assert call.norm(m=0, x=None) == 0 and ctx.launches == 0


def test_no_context_and_other_device(lib, call, ctx):
    none = Calls(lib, None)
    assert none.y() == none.dx() == none.dw() == none.lora() == none.norm() == -1
    ctx.current = 1
    assert call.y() == call.dx() == call.dw() == call.lora() == call.norm() == -1
    assert ctx.launches == 0


def test_every_launched_kernel_is_built(lib):
    """The kernels that any type, size and alignment selects are in the code objects, within the launch limits."""
    objects = b"".join(open(os.path.join(qmm.LIB_DIR, "le_qmm_%s.hsaco" % p), "rb").read() for p in PARTS)
    seen = set()

    def collect(f):
        c = Ctx()
        assert f(Calls(lib, c)) == 0, c.err
        assert c.launches <= 4
        fine(c)
        seen.update(name for name, _, _, _ in c.calls())

    sizes = (1, 7, 32, 64, 100, 256, 515, 1001, 1536, 2048, 4096, 28672)
    for ty in (0, 1, 30):
        for off in (0, 2 if ty else 4):
            for rows in sizes:
                for cols in sizes:
                    for n_exp, n_row in ((1, 1), (8, 16), (128, 64), (60, 300), (8, 4096), (1, 4096), (128, 32768), (1, 200000)):
                        kw = dict(ty=ty, x=A + off, rows=rows, cols=cols, ldx=cols, ldy=rows, n_exp=n_exp, n_row=n_row)
                        collect(lambda c: c.y(**kw))
                        collect(lambda c: c.dx(**kw))
                        collect(lambda c: c.dw(**kw))
                        collect(lambda c: c.dw(dwtype=0, **kw))
            for ltype in (0, 1, 30):
                for rank in (1, 4, 8, 12, 16, 31, 64, 100, 256):
                    for m in (1, 2, 15, 16, 61, 64, 65, 300, 4096):
                        for rows, cols in ((1, 1), (64, 4096), (4096, 64), (28672, 4096), (4096, 14336), (1001, 515)):
                            collect(lambda c: c.lora(xtype=ty, ltype=ltype, rank=rank, m=m, rows=rows, cols=cols, x=A + off, ldx=cols, ldb=rows, ldy=rows))
            for n in (32, 64, 96, 2048, 4096, 5120, 8192, 16384, 2**17):
                for m in (1, 37, 4096):
                    collect(lambda c: c.norm(ty=ty, n=n, m=m, x=A + off, ldx=n, ldr=n, ldh=n, ldo=n))
                    collect(lambda c: c.norm(ty=ty, n=n + 1, m=m, xq=None, xd=None, xs=None, ldx=n + 1, ldr=n + 1, ldh=n + 1, ldo=n + 1))
    assert len(seen) >= 20 and not [n for n in seen if (n + ".kd").encode() not in objects]


def test_python_adapters_refuse_other_tensors():
    import torch
    import lastengine_amd as le
    a, b, s = torch.zeros(3, 4, 32), torch.zeros(3, 16, 4), torch.zeros(3)
    assert le.Adapters(a, b, s, 3, 4, 16, 32).struct.ltype == le.F32 and le.Adapters(a, b, None, 3, 4, 16, 32).struct.scale is None
    for bad in ((a, b.half(), s, 3, 4, 16, 32), (a, b, s.half(), 3, 4, 16, 32), (a.double(), b.double(), s, 3, 4, 16, 32)):
        with pytest.raises(le.LeError) as e:
            le.Adapters(*bad)
        assert e.value.code == -2
    for bad in ((a, b, s, 3, 4, 16, 33), (a, b, s, 2, 4, 16, 32), (a, b, s[:2], 3, 4, 16, 32), (a.transpose(1, 2), b, s, 3, 4, 16, 32)):
        with pytest.raises(le.LeError) as e:
            le.Adapters(*bad)
        assert e.value.code == -3
