"""SwiGLU inside le_matvec_g4 where its rounding and range show: against the formula in 64 bits."""
import pytest

import lastengine_amd as le
from tests.test_gpu_g4 import run, torch_type

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ty", [le.F16, le.BF16])
def test_sixteen_bit_products_are_rounded(engine, ty):
    """One token of a 16-bit type: silu(gate) * up is held to 2^-16 of its value, to either side.

    A slot has two activations that are not zero, both with weight 1: a0 = silu(g) u, and a1 = -64 u' from a gate of 64 (silu(64) is 64
    in fp32), with u' the value of the type next to a0 / 64. So y = a0 + a1 is what u' is off by, at most 2^-8 a0, and shows
    a0's error. That is 2^-16 a0 for the two pieces; 2^-21 of a0 and of a1 (|a1| <= 1.01 |a0|) for silu; and for the sums (17 a0 + 17 a1 -
    16 (a0 + a1), in pieces): products of at most 17 a0, sums of activations of at most a0 that count 16 times, each rounded or
    aligned to 2^-24 of the largest term, for two pieces (the second 2^-7 of the first) no more than 2 * (17 + 16 * 1) * 2^-24 a0 * (1 + 2^-7) < 2^-17.9 a0.
    In all below (1 + 1 / 16 + 0.27) 2^-16 a0, and half a step of y. Pieces cut instead of rounded are off by up to 2^-15."""
    import torch
    slots, cols = 512, 32
    gen = torch.Generator().manual_seed(600)
    dt = torch_type(ty)
    g = (torch.rand(slots, generator=gen) * 6 + 2).to(dt).double()
    u = (torch.rand(slots, generator=gen) * 8 + 8).to(dt).double()
    a0 = g / (1 + (-g).exp()) * u
    u1 = -(a0 / 64).to(dt).double()
    x = torch.zeros(slots, 2 * cols, dtype=torch.float64)
    x[:, 5], x[:, cols + 5] = g, u
    x[:, 18], x[:, cols + 18] = 64.0, u1
    codes = torch.full((1, 1, cols // 2), 0x11, dtype=torch.uint8, device="cuda")
    one = torch.ones(1, 1, 1, dtype=torch.float16, device="cuda")
    w = le.G4(codes, one, torch.zeros_like(one), 1, cols, cols)
    out = torch.empty(slots, 1, 1, dtype=dt, device="cuda")
    sel = torch.zeros(slots, dtype=torch.int32, device="cuda")
    engine.mv_g4(ty, w, x.to(dt).cuda(), out, slots=slots, sel=sel, swiglu=True)
    want = a0 + 64 * u1
    err = (out.double().cpu().flatten() - want).abs()
    bound = (1 + 1 / 16 + 0.27) * 2.0 ** -16 * a0 + torch.finfo(dt).eps / 2 * want.abs()
    assert (want.abs() <= 2.0 ** -8 * a0 * 1.01).all()
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("ty", [le.F32, le.BF16])
@pytest.mark.parametrize("m", [1, 3, 20])
@pytest.mark.parametrize("gate", [-86.0, -87.5, -88.5, -92.0, -99.0, -104.0])
def test_far_gates_and_large_ups(engine, ty, m, gate):
    """Gates whose exponential fp32 does not hold, or not in full, beside ups so large that the product is an ordinary number.

    Activations lie between 2e38 and 3e38 times silu(gate +- 0.25), so all count alike. Their error, 2^-21 and 2^-16 or 2^-22 of the value, is
    below the bound's (cols + 8) 2^-24 times 47 of them; a product taken as 0 is off by all of it."""
    import torch
    cols = 256
    gen = torch.Generator().manual_seed(610)
    g = gate + torch.rand(m, cols, generator=gen) * 0.5 - 0.25
    u = (torch.rand(m, cols, generator=gen) * 1e38 + 2e38) * torch.where(torch.rand(m, cols, generator=gen) < 0.5, -1.0, 1.0)
    x = torch.cat([g, u], 1).to(torch_type(ty))
    run(engine, ty, le.F16, 1, 40, cols, 64, m, 1, 1, None, True, True, 611, x=x, rms=False)
