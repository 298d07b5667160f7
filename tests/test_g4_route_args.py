"""Argument checks and launch shapes of le_matvec_g4 and of the expert-routing entries, without a GPU: their host sources are
compiled against a context whose launches are only written down."""
import ctypes
import os
import shutil
import subprocess

import pytest

from lastengine_amd import build, qmm
from tests.conftest import REPO

STUB = r"""
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include "le_ctx.h"
struct le_ctx { char err[512]; int device, current; int launches; char name[4][64]; unsigned g[4][3]; int block[4]; unsigned long lds[4]; };
int le_ctx_device(const le_ctx *c) { return c->device; }
int le_ctx_cus(const le_ctx *) { return 256; }
int le_ctx_fail(le_ctx *c, int code, const char *msg) { return le_ctx_failf(c, code, "%s", msg); }
int le_ctx_failf(le_ctx *c, int code, const char *fmt, ...) { va_list ap; va_start(ap, fmt); vsnprintf(c->err, sizeof c->err, fmt, ap); va_end(ap); return code; }
int le_ctx_on_device(le_ctx *c) { return c->device == c->current ? LE_OK : le_ctx_failf(c, LE_ERR_ARG, "device"); }
int le_ctx_launch(le_ctx *c, const char *name, dim3 g, int block, size_t lds, hipStream_t, void **) {
    const int i = c->launches++ & 3;
    snprintf(c->name[i], 64, "%s", name);
    c->g[i][0] = g.x, c->g[i][1] = g.y, c->g[i][2] = g.z, c->block[i] = block, c->lds[i] = lds;
    return LE_OK;
}
"""


class Ctx(ctypes.Structure):
    _fields_ = [("err", ctypes.c_char * 512), ("device", ctypes.c_int), ("current", ctypes.c_int), ("launches", ctypes.c_int),
                ("name", (ctypes.c_char * 64) * 4), ("g", (ctypes.c_uint * 3) * 4), ("block", ctypes.c_int * 4),
                ("lds", ctypes.c_ulong * 4)]

    def calls(self):
        return [(self.name[i].value.decode(), tuple(self.g[i]), self.block[i], self.lds[i]) for i in range(min(self.launches, 4))]


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if not shutil.which("g++") or not os.path.exists(os.path.join(build.ROCM, "include", "hip", "hip_runtime.h")):
        pytest.skip("no g++ or HIP headers")
    d = tmp_path_factory.mktemp("args")
    (d / "stub.cpp").write_text(STUB)
    so = str(d / "libargs.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I" + build.ROCM + "/include", "-I" + build.CSRC,
                    "-I" + os.path.join(REPO, "include"), str(d / "stub.cpp")] + [os.path.join(build.CSRC, f) for f in ("le_g4.cpp", "le_route.cpp")] +
                   ["-o", so], check=True)
    L, real = ctypes.CDLL(so), qmm.lib()
    for name in ("le_matvec_g4", "le_matvec_g4_workspace_size", "le_moe_route", "le_moe_route_bwd", "le_moe_sort", "le_moe_sort_workspace_size", "le_moe_permute", "le_moe_combine",
                 "le_moe_combine_bwd"):
        getattr(L, name).restype, getattr(L, name).argtypes = getattr(real, name).restype, getattr(real, name).argtypes
    return L


@pytest.fixture
def ctx():
    return Ctx()


A = 0x10000  # an aligned address; nothing is read there


def g4(L, c, codes=A, scales=A, zeros=A, n_mat=4, rows=64, cols=256, group=64, stype=1, sel=A, slots=2, share=1, xtype=0, x=A, xstride=256, m=1,
       y=A, swiglu=0, w=True, ws=A, ws_bytes=1 << 40):
    s = qmm._G4(codes, scales, zeros, n_mat, rows, cols, group, stype)
    return L.le_matvec_g4(ctypes.addressof(c), ctypes.addressof(s) if w else None, sel, slots, share, xtype, x, xstride, m, y, swiglu, ws, ws_bytes, None)


@pytest.mark.parametrize("bad,code", [
    (dict(w=False), -1), (dict(codes=None), -1), (dict(scales=None), -1), (dict(x=None), -1), (dict(y=None), -1),
    (dict(xtype=8), -2), (dict(stype=12), -2), (dict(xtype=-1), -2),
    (dict(rows=0), -3), (dict(cols=0), -3), (dict(n_mat=0), -3), (dict(slots=0), -3), (dict(share=0), -3), (dict(m=0), -3), (dict(m=65), -3),
    (dict(rows=-5), -3), (dict(slots=65536), -3), (dict(cols=250, group=250), -3), (dict(cols=48, group=48), -3), (dict(group=16), -3),
    (dict(group=96, cols=192), -3), (dict(group=512), -3), (dict(group=0), -3), (dict(group=-64), -3), (dict(sel=None, slots=5), -3),
    (dict(xstride=255), -3), (dict(xstride=-256), -3), (dict(swiglu=1, xstride=256), -3), (dict(rows=2**31 - 1, n_mat=1), -3), (dict(rows=2**25, n_mat=1), -3), (dict(cols=2**25, group=2**25, xstride=2**25), -3),
    (dict(rows=2**28, cols=32, group=32, stype=0), -3), (dict(rows=2**28, cols=32, group=32), -3), (dict(m=2, slots=40000, n_mat=40000, sel=None), -3),
    (dict(m=2, ws=None), -7), (dict(m=2, ws_bytes=2 * 256 * 2), -7), (dict(m=5, xtype=30, ws=None), -7), (dict(m=2, swiglu=1, xstride=512, ws_bytes=99), -7),
    (dict(m=2, ws=A + 8), -4),
    (dict(codes=A + 8), -4), (dict(x=A + 4), -4), (dict(xstride=258), -4), (dict(xtype=1, xstride=260), -4), (dict(scales=A + 1), -4),
    (dict(zeros=A + 1), -4), (dict(stype=0, scales=A + 2), -4), (dict(y=A + 2), -4), (dict(sel=A + 2), -4)])
def test_g4_refusals(lib, ctx, bad, code):
    assert g4(lib, ctx, **bad) == code
    assert ctx.launches == 0 and ctx.err
    assert lib.le_matvec_g4(None, None, None, 1, 1, 0, None, 0, 1, None, 0, None, 0, None) == -1


def test_every_launched_kernel_is_built(lib):
    """The kernels that any type, group and number of tokens selects are in the code objects, within the launch limits."""
    objects = b"".join(open(os.path.join(qmm.LIB_DIR, "le_qmm_%s.hsaco" % p), "rb").read() for p in ("g4s0", "g4s1", "g4s30", "rt"))
    seen = set()

    def collect(c):
        for name, g, block, lds in c.calls():
            assert g[0] * block < 2**32 and g[1] <= 65535 and g[2] <= 65535 and min(g) > 0 and block <= 1024 and lds <= 160 * 1024, (name, g, block, lds)
            seen.add(name)

    for xtype in (0, 1, 30):
        for stype in (0, 1, 30):
            for swiglu in (0, 1):
                for cols, group in ((32, 32), (4096, 32), (9216, 32), (4160, 64), (9216, 64), (4096, 128), (12288 + 128, 128), (4000, 4000), (65536, 256)):
                    for m in (1, 2, 3, 4, 5, 6, 7, 8, 9, 16, 17, 64):
                        c = Ctx()
                        assert g4(lib, c, xtype=xtype, stype=stype, swiglu=swiglu, cols=cols, group=group, xstride=cols * (1 + swiglu), m=m, rows=5000) == 0
                        collect(c)
        for n_tok in (1, 5000):
            for n_exp in (1, 32, 64, 128, 256, 500, 1024):
                c = Ctx()
                assert lib.le_moe_route(ctypes.addressof(c), xtype, A, n_tok, n_exp, 1, A, A, None) == 0
                assert lib.le_moe_route_bwd(ctypes.addressof(c), xtype, A, A, A, n_tok, n_exp, 1, A, None) == 0
                assert lib.le_moe_sort(ctypes.addressof(c), A, n_tok, 4, n_exp, A, A, A, A, A, 1 << 30, None) == 0
                collect(c)
            for cols, ld in ((8, 8), (100, 104), (256, 256), (2048, 2048), (2047, 2047), (100000, 100000)):
                c, k = Ctx(), 4
                assert lib.le_moe_permute(ctypes.addressof(c), xtype, A, ld, A, n_tok, k, cols, A, ld, 9, None) == 0
                assert lib.le_moe_combine(ctypes.addressof(c), xtype, A, ld, 9, A, A, n_tok, k, cols, A, ld, None) == 0
                assert lib.le_moe_combine_bwd(ctypes.addressof(c), xtype, A, ld, A, ld, 9, A, A, n_tok, k, cols, A, A, None) == 0
                collect(c)
    assert len(seen) > 100 and not [n for n in seen if (n + ".kd").encode() not in objects]


@pytest.mark.parametrize("good", [
    dict(), dict(zeros=None), dict(sel=None), dict(xstride=0), dict(group=256), dict(cols=96, group=96), dict(cols=96, group=32), dict(cols=32, group=32),
    dict(m=64), dict(slots=65535), dict(swiglu=1, xstride=512), dict(xtype=30, stype=30, y=A + 2, scales=A + 2), dict(rows=1), dict(rows=2**24, n_mat=1), dict(m=4, xtype=30, ws=None), dict(m=2, xtype=1, ws=None), dict(m=64, cols=2**20, group=2**20, xstride=2**20), dict(m=17, slots=900, cols=14336, xstride=14336),
    dict(cols=2**20, group=2**20, xstride=2**20)])
def test_g4_launches(lib, ctx, good):
    assert g4(lib, ctx, **good) == 0, ctx.err
    assert 1 <= ctx.launches <= 3
    for name, g, block, lds in ctx.calls():
        assert g[0] * block < 2**32 and g[1] <= 65535 and g[2] <= 65535 and min(g) > 0 and lds <= 160 * 1024, (name, g, block, lds)


def test_g4_workspace(lib):
    def f(xtype, m, cols, slots, share, swiglu, rows=64, group=64, w=True):
        s = qmm._G4(A, A, A, 4, rows, cols, group, 1)
        return lib.le_matvec_g4_workspace_size(ctypes.addressof(s) if w else None, xtype, m, slots, share, swiglu)

    assert f(0, 1, 4096, 8, 1, 1) == 0 and f(30, 4, 4096, 1, 1, 0) == 0 and f(1, 2, 4096, 1, 1, 0) == 0  # one launch
    assert f(30, 2, 4096, 1, 1, 1) >= 2 * 4096 * 4
    assert f(0, 2, 4096, 1, 1, 0) >= 2 * 4096 * 4 and f(30, 5, 4096, 1, 1, 0) >= 5 * 4096 * 2 and f(1, 3, 4096, 1, 1, 0) >= 3 * 4096 * 2
    assert f(0, 2, 4096, 8, 2, 0) == 4 * f(0, 2, 4096, 1, 1, 0)  # sets of activations
    assert f(0, 2, 14336, 3, 1, 0, rows=128) >= 3 * 2 * 14336 * 4 + 4 * 3 * 2 * 128 * 4  # and the partial results of K's segments
    assert f(0, 2, 4096, 3, 1, 0, rows=128, group=32) >= 3 * 2 * 4096 * 4 + 2 * 3 * 2 * 128 * 4
    for bad in ((8, 2, 4096, 1, 1, 0), (0, 0, 4096, 1, 1, 0), (0, 65, 4096, 1, 1, 0), (0, 2, 100, 1, 1, 0), (0, 2, 4096, 0, 1, 0), (0, 2, 4096, 1, 0, 0)):
        assert f(*bad) == 0
    assert f(0, 2, 4096, 1, 1, 0, w=False) == 0


def test_other_device(lib, ctx):
    ctx.current = 1
    c = ctypes.addressof(ctx)
    assert g4(lib, ctx) == -1
    assert lib.le_moe_route(c, 0, A, 4, 8, 2, A, A, None) == -1
    assert lib.le_moe_sort(c, A, 4, 2, 8, A, A, A, A, A, 1 << 20, None) == -1
    assert lib.le_moe_permute(c, 0, A, 8, A, 4, 2, 8, A, 8, 8, None) == -1
    assert ctx.launches == 0


def test_route_refusals(lib, ctx):
    c = ctypes.addressof(ctx)

    def route(ltype=0, logits=A, n_tok=4, n_exp=8, k=2, idx=A, w=A):
        return lib.le_moe_route(c, ltype, logits, n_tok, n_exp, k, idx, w, None)

    def bwd(ltype=0, idx=A, w=A, dw=A, n_tok=4, n_exp=8, k=2, dl=A):
        return lib.le_moe_route_bwd(c, ltype, idx, w, dw, n_tok, n_exp, k, dl, None)

    for f in (route, bwd):
        assert f(ltype=12) == -2
        for bad in (dict(n_tok=-1), dict(k=0), dict(k=17, n_exp=32), dict(k=9), dict(n_exp=0), dict(n_exp=1025), dict(n_tok=2**30)):
            assert f(**bad) == -3, bad
        assert f(idx=None) == -1 and f(w=None) == -1
        assert f(idx=A + 2) == -4 and f(w=A + 1) == -4
        assert f(n_tok=0) == 0
    assert route(logits=None) == -1 and route(logits=A + 2) == -4 and route(ltype=30, logits=A + 1) == -4
    assert bwd(dw=None) == -1 and bwd(dl=None) == -1 and bwd(dl=A + 2) == -4 and bwd(dw=A + 1) == -4
    assert ctx.launches == 0
    assert route() == 0 and bwd() == 0 and route(ltype=1, logits=A + 2) == 0
    assert lib.le_moe_route(None, 0, A, 4, 8, 2, A, A, None) == -1 and lib.le_moe_route_bwd(None, 0, A, A, A, 4, 8, 2, A, None) == -1


def test_sort_refusals(lib, ctx):
    c = ctypes.addressof(ctx)

    def sort(idx=A, n_tok=4, k=2, n_exp=8, off=A, i=A, o=A, pos=A, ws=A, ws_bytes=1 << 30):
        return lib.le_moe_sort(c, idx, n_tok, k, n_exp, off, i, o, pos, ws, ws_bytes, None)

    for bad in (dict(n_tok=-1), dict(k=0), dict(k=17), dict(n_exp=0), dict(n_exp=1025), dict(n_tok=2**28, k=16)):
        assert sort(**bad) == -3, bad
    assert sort(idx=None) == -1 and sort(off=None) == -1
    for bad in (dict(idx=A + 2), dict(off=A + 1), dict(i=A + 2), dict(o=A + 2), dict(pos=A + 2), dict(ws=A + 8)):
        assert sort(**bad) == -4, bad
    big = lib.le_moe_sort_workspace_size(65536, 8, 128)
    if big:
        assert sort(n_tok=65536, k=8, n_exp=128, ws_bytes=big - 1) == -7 and sort(n_tok=65536, k=8, n_exp=128, ws=None) == -7
    assert lib.le_moe_sort_workspace_size(1, 8, 128) == 0  # a decoded token needs none
    assert lib.le_moe_sort_workspace_size(-1, 8, 128) == 0 and lib.le_moe_sort_workspace_size(4, 17, 128) == 0
    assert ctx.launches == 0
    assert sort() == 0 and sort(idx=None, n_tok=0) == 0 and sort(i=None, o=None, pos=None) == 0
    assert sort(n_tok=65536, k=8, n_exp=128, ws_bytes=big) == 0 and sort(n_tok=2**27 - 1, k=16) == 0
    for name, g, block, lds in ctx.calls():
        assert g[0] * block < 2**32 and min(g) > 0 and lds <= 160 * 1024
    assert lib.le_moe_sort(None, A, 4, 2, 8, A, A, A, A, A, 0, None) == -1


def test_rows_refusals(lib, ctx):
    c = ctypes.addressof(ctx)

    def permute(ty=0, x=A, ldt=8, pos=A, n_tok=4, k=2, cols=8, e=A, lde=8, n_row=8, w=A):
        return lib.le_moe_permute(c, ty, x, ldt, pos, n_tok, k, cols, e, lde, n_row, None)

    def combine(ty=0, x=A, ldt=8, pos=A, n_tok=4, k=2, cols=8, e=A, lde=8, n_row=8, w=A):
        return lib.le_moe_combine(c, ty, e, lde, n_row, pos, w, n_tok, k, cols, x, ldt, None)

    def bwd(ty=0, x=A, ldt=8, pos=A, n_tok=4, k=2, cols=8, e=A, lde=8, n_row=8, w=A, de=A, dw=A):
        return lib.le_moe_combine_bwd(c, ty, x, ldt, e, lde, n_row, pos, w, n_tok, k, cols, de, dw, None)

    for f in (permute, combine, bwd):
        assert f(ty=8) == -2
        for bad in (dict(n_tok=-1), dict(k=0), dict(k=17), dict(cols=0), dict(cols=2**25 + 1, ldt=2**26, lde=2**26), dict(cols=2**31 - 1, ldt=2**31, lde=2**31), dict(n_row=-1), dict(ldt=7), dict(lde=7), dict(n_tok=2**31 - 1)):
            assert f(**bad) == -3, bad
        assert f(x=None) == -1 and f(e=None) == -1
        assert f(x=A + 2) == -4 and f(e=A + 2) == -4 and f(ty=1, x=A + 1) == -4 and f(pos=A + 2) == -4
        assert f(n_tok=0) == 0
    assert combine(w=A + 2) == -4 and bwd(w=A + 2) == -4 and bwd(de=A + 1) == -4 and bwd(dw=A + 2) == -4
    assert permute(n_row=0) == 0 and bwd(de=None, dw=None) == 0
    assert ctx.launches == 0
    for f in (permute, combine, bwd):
        assert f() == 0 and f(pos=None) == 0 and f(cols=2**25, ldt=2**25, lde=2**25) == 0 and f(ty=30, x=A + 2, e=A + 2) == 0 and f(n_tok=2**27, k=1) == 0
    assert bwd(dw=None, e=None) == 0 and bwd(de=None) == 0 and combine(w=None) == 0 and combine(e=None, n_row=0) == 0
    for name, g, block, lds in ctx.calls():
        assert g[0] * block < 2**32 and g[1] <= 65535 and min(g) > 0 and lds <= 160 * 1024, (name, g, block)
    assert lib.le_moe_permute(None, 0, A, 8, A, 4, 2, 8, A, 8, 8, None) == -1
    assert lib.le_moe_combine(None, 0, A, 8, 8, A, A, 4, 2, 8, A, 8, None) == -1
    assert lib.le_moe_combine_bwd(None, 0, A, 8, A, 8, 8, A, A, 4, 2, 8, A, A, None) == -1
