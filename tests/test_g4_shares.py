"""How le_matvec_g4 shares row groups out to blocks, without a GPU: the host source compiled against a context that keeps the arguments of its
launches."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

from lastengine_amd import build, qmm
from tests.conftest import REPO
from tests.test_gpu_g4_groups import CASES, N_MAT

STUB = r"""
#include <cstdio>
#include <cstring>
#include "le_ctx.h"
#include "le_g4_args.h"
struct le_ctx { int launches; struct { char name[48]; unsigned g[3]; int block; unsigned long lds; int gx, per, full, nw, segs; } l[3]; };
int le_ctx_device(const le_ctx *) { return 0; }
int le_ctx_cus(const le_ctx *) { return 256; }
int le_ctx_fail(le_ctx *, int code, const char *) { return code; }
int le_ctx_failf(le_ctx *, int code, const char *, ...) { return code; }
int le_ctx_on_device(le_ctx *) { return LE_OK; }
int le_ctx_launch(le_ctx *c, const char *name, dim3 g, int block, size_t lds, hipStream_t, void **args) {
    const G4Args &a = *(const G4Args *)args[0];
    auto &l = c->l[c->launches++];
    snprintf(l.name, sizeof l.name, "%s", name);
    l.g[0] = g.x, l.g[1] = g.y, l.g[2] = g.z, l.block = block, l.lds = lds;
    l.gx = a.gx, l.per = a.per, l.full = a.full, l.nw = a.nw, l.segs = a.segs;
    return LE_OK;
}
"""
A = 0x10000  # an aligned address; nothing is read there


class Launch(ctypes.Structure):
    _fields_ = [("name", ctypes.c_char * 48), ("g", ctypes.c_uint * 3), ("block", ctypes.c_int), ("lds", ctypes.c_ulong), ("gx", ctypes.c_int),
                ("per", ctypes.c_int), ("full", ctypes.c_int), ("nw", ctypes.c_int), ("segs", ctypes.c_int)]


class Ctx(ctypes.Structure):
    _fields_ = [("launches", ctypes.c_int), ("l", Launch * 3)]


@pytest.fixture(scope="module")
def product(tmp_path_factory):
    """The launch of the product itself, of a call's one to three."""
    if not shutil.which("g++") or not os.path.exists(os.path.join(build.ROCM, "include", "hip", "hip_runtime.h")):
        pytest.skip("no g++ or HIP headers")
    d = tmp_path_factory.mktemp("shares")
    (d / "stub.cpp").write_text(STUB)
    so = str(d / "libshares.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I" + build.ROCM + "/include", "-I" + build.CSRC,
                    "-I" + os.path.join(REPO, "include"), str(d / "stub.cpp"), os.path.join(build.CSRC, "le_g4.cpp"), "-o", so], check=True)
    L, real = ctypes.CDLL(so), qmm.lib()
    L.le_matvec_g4.restype, L.le_matvec_g4.argtypes = real.le_matvec_g4.restype, real.le_matvec_g4.argtypes

    def call(xtype, stype, zeros, rows, cols, group, m, slots, share, swiglu):
        c, w = Ctx(), qmm._G4(A, A, A if zeros else None, N_MAT, rows, cols, group, stype)
        width = cols * (1 + swiglu)
        assert L.le_matvec_g4(ctypes.addressof(c), ctypes.addressof(w), A, slots, share, xtype, A, width, m, A, int(swiglu), A, 1 << 62, None) == 0
        at = [i for i in range(c.launches) if c.l[i].name[:6] in (b"le_g4q", b"le_g4t", b"le_g4m")]
        assert len(at) == 1
        return c.l[at[0]]
    return call


@pytest.mark.parametrize("case", CASES, ids=lambda c: c[0])
def test_cases_have_several_row_groups(product, case):
    rows = case[4]
    l = product(*case[1:])
    assert l.name.decode() == case[0]
    assert l.per >= 3 and 0 < l.full < l.gx and rows % 16, (l.per, l.full, l.gx)


def test_cases_cover_the_kernels():
    """Every kind of kernel, scale block and type is among them."""
    names = [c[0] for c in CASES]
    for kind in ("f32", "f16", "bf16", "f32w", "f16w", "bf16w", "f16t2", "bf16t4"):
        for form in ("_s", "_mp_s"):
            mine = [n for n in names if n.startswith("le_g4q_%s_" % kind) and ("_mp" in n) == (form == "_mp_s")]
            assert mine or (kind, form) == ("f16w", "_mp_s"), (kind, form)
    for kind in ("n1_p1", "n1_p2", "n2_p1", "n2_p2", "n3_p2"):
        assert any(n.startswith("le_g4t_" + kind) for n in names)
    for block in ("b32", "b64", "b128"):
        for kind in ("le_g4q", "le_g4t", "le_g4m_p1", "le_g4m_p2"):
            assert any(n.startswith(kind) and block in n for n in names), (kind, block)


def test_blocks_take_each_group_once(product):
    """Over shapes of all kinds: the groups of a slot's blocks, as the kernels number them, are all of the rows' and no two the same, and a block's
    partial results fit its LDS."""
    rng = random.Random(7)
    most = 0
    for _ in range(4000):
        group = rng.choice([32, 64, 128, 256])
        cols = group * rng.choice([1, 2, 7, 16, 33, 64, 112, 300])
        rows = int(2 ** rng.uniform(0, 17)) + rng.randrange(16)
        m, slots, share, swiglu = rng.choice([1, 1, 2, 3, 4, 5, 6, 8, 9, 16, 17, 40, 64]), rng.choice([1, 1, 2, 3, 8, 32, 200, 900]), rng.choice([1, 2, 8]), rng.random() < 0.3
        if slots * m * rows > 1 << 31 or rows * cols >= 1 << 33:
            continue
        l = product(rng.choice([0, 1, 30]), 1, True, rows, cols, group, m, slots, share, swiglu)
        groups = (rows + 15) // 16
        assert l.g[0] == l.gx and l.g[1] == slots and l.block == 64 * l.nw <= 1024 and l.lds <= 160 * 1024
        assert 0 < l.full <= l.gx
        # block b takes b, b + gx, ..: per of them, blocks from `full` on one less
        assert l.per >= 1 and (l.per - 1) * l.gx + l.full == groups
        most = max(most, l.per)
        name = l.name.decode()
        if name.startswith("le_g4m"):
            each = 1024
        elif name.startswith("le_g4t"):
            each = int(name[8]) * (4 // int(name[11])) * 256  # sets of four rows, pieces of a token
        else:
            each = 256 * (2 if "t2" in name else 4 if "t4" in name else 1)
        fixed = l.nw * 4096 if name.startswith("le_g4q") and not ("_bf16_" in name or "t2" in name or "t4" in name) else 0
        assert l.lds == fixed + l.per * l.nw * each, name
    assert most >= 8
