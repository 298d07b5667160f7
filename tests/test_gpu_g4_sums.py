"""What the sums of le_matvec_g4 are off by where activations differ far in size, against 64 bits.

With u = 2^-24 and T = the sum over c of |scale| (31 + 16 + |zero|) |a| of an output: every product, of at most that term, meets on its way to the output at
most 128 additions inside its scale block, then (4096 columns) 3 over pieces, the product with the scale, 16 over the blocks of a lane, 2 over lanes and 16
over waves, 2 over segments, each off by u of a sum that is at most T; 4 more are the 2^-22 that an activation may be off by. In all less than 128 + 48."""
import pytest

import lastengine_amd as le
from tests.test_gpu_g4 import U, dequant, make, torch_type

pytestmark = pytest.mark.gpu

ROWS, COLS = 200, 4096


def run(engine, ty, codes, scales, z, group, x):
    import torch
    w = le.G4(codes.cuda(), scales.cuda(), z.cuda() if z is not None else None, ROWS, COLS, group)
    out = torch.full((len(x), ROWS), float("nan"), dtype=torch_type(ty), device="cuda")
    engine.mv_g4(ty, w, x.cuda(), out, m=len(x))
    wf, mag = dequant(codes, scales, z, group)
    a = x.double()
    return out.double().cpu(), a @ wf[0].t(), a.abs() @ mag[0].t()


def check(out, want, terms, ty):
    import torch
    half = 0.0 if ty == le.F32 else torch.finfo(torch_type(ty)).eps / 2
    err, bound = (out - want).abs(), half * want.abs() + (1 + half) * (128 + 48) * U * terms
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("ty", [le.F32, le.F16, le.BF16])
@pytest.mark.parametrize("m", [1, 2, 5, 20])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_large_activations_that_meet_weight_zero(engine, ty, m, group, zeros):
    """Eight channels of 1000 whose codes equal the zero point: they add nothing to an output but their rounding."""
    import torch
    codes, scales, z = make(1, ROWS, COLS, group, le.F16, False, 800)
    big = torch.randperm(COLS // 2, generator=torch.Generator().manual_seed(801))[:8]
    codes[..., big] = 0x88
    z = torch.full_like(scales, 8.0) if zeros else None
    x = torch.randn(m, COLS, generator=torch.Generator().manual_seed(802))
    x[:, 2 * big] = 1000.0
    check(*run(engine, ty, codes, scales, z, group, x.to(torch_type(ty))), ty)


@pytest.mark.parametrize("ty", [le.F32, le.BF16])
@pytest.mark.parametrize("m", [1, 2, 5, 20])
@pytest.mark.parametrize("exponent", [114, -100])
def test_largest_and_small_activations(engine, ty, m, exponent):
    """As large as sums of (16 + code) a leave room for: 128 columns of |a| sum to less than 256 * 2^114, and 31 times that is below 2^127."""
    import torch
    codes, scales, z = make(1, ROWS, COLS, 64, le.F16, True, 810, frac=True)
    x = torch.randn(m, COLS, generator=torch.Generator().manual_seed(811))
    assert float(x.abs().reshape(m, -1, 128).sum(-1).max()) < 256
    check(*run(engine, ty, codes, scales, z, 64, (x * 2.0 ** exponent).to(torch_type(ty))), ty)
