"""le_matvec_g4 where a block goes over several groups of 16 rows, as it does at the sizes of real matrices: the loads that run ahead, the
partial results of each group, blocks with one group less than others, rows that end inside the last group.

Every output is compared with a plain form in 64 bits on the device; what is compared, and its tolerance, are those of
test_gpu_g4.py. test_g4_shares.py holds (without a GPU) that each case here runs the kernel it names, with at least three row groups in some
blocks and one fewer in others."""
import pytest

import lastengine_amd as le
from tests.test_gpu_g4 import check, make, torch_type

F32, F16, BF16 = le.F32, le.F16, le.BF16

# kernel: activations, scales, zero points?, rows, cols, group, tokens, slots, share, SwiGLU?
CASES = [
    # one launch, K in one pass (4 or 8 waves)
    ("le_g4q_f32_b128_s1", F32, F16, True, 2067, 2048, 128, 1, 24, 1, False),
    ("le_g4q_f32_b64v_s0", F32, F32, True, 1107, 4096, 64, 1, 22, 1, False),
    ("le_g4q_f32_b32_s30", F32, BF16, False, 1107, 4000, 32, 1, 15, 1, False),
    ("le_g4q_f16_b32v_s1", F16, F16, True, 2067, 2048, 32, 1, 35, 8, False),
    ("le_g4q_f16_b64_s1", F16, F16, False, 1107, 3648, 64, 1, 15, 3, False),
    ("le_g4q_bf16_b128_s30", BF16, BF16, False, 1107, 3744, 3744, 1, 22, 1, False),
    ("le_g4q_bf16_b32v_s1", BF16, F16, True, 1107, 4096, 32, 1, 22, 1, False),
    ("le_g4q_f32w_b64v_s1", F32, F16, True, 1107, 4096, 64, 1, 22, 1, True),
    ("le_g4q_f16w_b32v_s1", F16, F16, False, 2067, 768, 32, 1, 48, 1, True),
    ("le_g4q_bf16w_b128_s1", BF16, F16, True, 1107, 4096, 256, 1, 22, 1, True),
    ("le_g4q_f16t2_b64v_s1", F16, F16, True, 1107, 4096, 64, 2, 15, 1, False),
    ("le_g4q_f16t2_b32_s0", F16, F32, True, 1107, 3616, 32, 2, 22, 2, False),
    ("le_g4q_bf16t4_b128_s1", BF16, F16, True, 1107, 4096, 128, 4, 15, 1, False),
    ("le_g4q_bf16t4_b32v_s1", BF16, F16, False, 1089, 4096, 32, 3, 29, 1, False),
    # ... in several, or with more waves
    ("le_g4q_f32_b128_mp_s1", F32, F16, True, 1026, 9216, 128, 1, 8, 1, False),
    ("le_g4q_f32_b32v_mp_s1", F32, F16, False, 1107, 14336, 32, 1, 11, 1, False),
    ("le_g4q_f16_b64_mp_s1", F16, F16, True, 1026, 9152, 64, 1, 8, 1, False),
    ("le_g4q_bf16_b32_mp_s30", BF16, BF16, True, 1107, 8608, 32, 1, 11, 1, False),
    ("le_g4q_f32w_b64v_mp_s1", F32, F16, True, 1026, 14336, 64, 1, 8, 1, True),
    ("le_g4q_bf16w_b128_mp_s1", BF16, F16, False, 1107, 14464, 128, 1, 11, 1, True),
    ("le_g4q_f16t2_b32v_mp_s1", F16, F16, True, 1107, 8448, 32, 2, 22, 1, False),
    ("le_g4q_bf16t4_b64v_mp_s1", BF16, F16, True, 1107, 9216, 64, 4, 11, 1, False),
    # sets of four virtual rows from the workspace, K in one segment or several
    ("le_g4t_n1_p2_b128_s1", F32, F16, True, 1026, 4096, 128, 2, 8, 1, False),
    ("le_g4t_n1_p1_b32_s1", F16, F16, False, 1107, 4000, 32, 3, 11, 1, False),
    ("le_g4t_n2_p1_b64v_s1", BF16, F16, True, 1026, 4096, 64, 8, 8, 1, False),
    ("le_g4t_n2_p1_b64v_w_s1", BF16, F16, True, 1107, 5120, 64, 6, 11, 1, False),
    ("le_g4t_n2_p2_b32v_s0", F32, F32, True, 1026, 4096, 32, 4, 8, 2, False),
    ("le_g4t_n2_p2_b64_s1", F32, F16, False, 1041, 14272, 64, 3, 8, 1, True),
    ("le_g4t_n3_p2_b64v_s1", F32, F16, True, 4077, 14336, 64, 5, 1, 1, True),
    ("le_g4t_n3_p2_b128_s30", F16, BF16, True, 1026, 6272, 128, 6, 6, 1, True),
    ("le_g4t_n3_p2_b32_s1", F32, F16, True, 1026, 4128, 32, 5, 4, 1, False),
    # tiles of 16 tokens
    ("le_g4m_p1_b128_s1", BF16, F16, True, 1107, 4096, 128, 16, 11, 1, False),
    ("le_g4m_p1_b32_s1", F16, F16, False, 1026, 2080, 32, 9, 8, 1, False),
    ("le_g4m_p1_b64v_s1", BF16, F16, True, 1026, 6144, 64, 33, 2, 1, False),
    ("le_g4m_p2_b32v_s1", F32, F16, True, 1026, 4096, 32, 20, 3, 1, False),
    ("le_g4m_p2_b64_s0", F32, F32, False, 1002, 4160, 64, 64, 2, 1, False),
    ("le_g4m_p2_b128_s1", F32, F16, True, 4077, 14336, 256, 17, 1, 1, True),
]
N_MAT = 3


def selection(slots):
    """Matrices of a stack of three for many slots, one of them outside it (no output but zeros), or the stack's first."""
    return [(5 * s + 1) % N_MAT for s in range(slots - 1)] + [-1] if slots > 1 else [2]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: c[0])
def test_several_row_groups_a_block(engine, case):
    import torch
    name, ty, stype, zeros, rows, cols, group, m, slots, share, swiglu = case
    print(case, flush=True)
    codes, scales, z = make(N_MAT, rows, cols, group, stype, zeros, 700 + rows + cols)
    codes, scales, z = codes.cuda(), scales.cuda(), z.cuda() if zeros else None
    w = le.G4(codes, scales, z, rows, cols, group, n_mat=N_MAT)
    width = cols * (1 + swiglu)
    x = torch.randn(-(-slots // share) * m, width, generator=torch.Generator().manual_seed(701)).to(torch_type(ty))
    n = slots * m * rows
    out = torch.full((n + 64,), 77.0, dtype=torch_type(ty), device="cuda")
    sel = selection(slots)
    engine.mv_g4(ty, w, x.cuda(), out, m=m, slots=slots, share=share, sel=torch.tensor(sel, dtype=torch.int32).cuda(), swiglu=swiglu)
    torch.cuda.synchronize()
    assert (out[n:] == 77.0).all(), "written behind the last output"
    got = out[:n].reshape(slots, m, rows)
    a = x.cuda().double()
    a = (a[:, :cols] / (1 + (-a[:, :cols]).exp()) * a[:, cols:] if swiglu else a).reshape(-1, m, cols)
    for mat in range(N_MAT):  # one matrix at a time in 64 bits
        slots_of = [s for s in range(slots) if sel[s] == mat]
        if not slots_of:
            continue
        q = torch.stack([codes[mat] & 15, codes[mat] >> 4], -1).flatten(-2).double()
        s64 = scales[mat].double().repeat_interleave(group, -1)
        zz = z[mat].double().repeat_interleave(group, -1) if zeros else torch.full_like(q, 8.0)
        wf, mag = ((q - zz) * s64).t().contiguous(), ((47 + zz.abs()) * s64.abs()).t().contiguous()
        for s in slots_of:
            act = a[s // share]
            check(got[s], (act @ wf).cpu(), (act.abs() @ mag).cpu(), ty, cols)
    for s in range(slots):
        assert sel[s] >= 0 or (got[s] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("case", [c for c in CASES if c[0][:6] in ("le_g4t", "le_g4m")][::2] + CASES[:2], ids=lambda c: c[0])
def test_same_bits_whatever_the_workspace_held(engine, case):
    """Sums in a fixed order: equal bits from call to call, with nothing read from the workspace that the call has not written, on blocks of
    several row groups and K in one segment or several."""
    import torch
    name, ty, stype, zeros, rows, cols, group, m, slots, share, swiglu = case
    print(case, flush=True)
    codes, scales, z = make(N_MAT, rows, cols, group, stype, zeros, 720 + rows)
    w = le.G4(codes.cuda(), scales.cuda(), z.cuda() if zeros else None, rows, cols, group, n_mat=N_MAT)
    x = torch.randn(-(-slots // share) * m, cols * (1 + swiglu), generator=torch.Generator().manual_seed(721)).to(torch_type(ty)).cuda()
    sel = torch.tensor(selection(slots), dtype=torch.int32).cuda()
    need = engine.mv_g4_workspace_size(ty, w, m, slots, share, swiglu)
    outs = []
    for fill in (0x00, 0xFF, 0x7C, 0x3F):  # zeros, NaN, fp16 and fp32 of ordinary and large size
        ws = torch.full((need,), fill, dtype=torch.uint8, device="cuda") if need else None
        out = torch.full((slots, m, rows), float("nan"), dtype=torch_type(ty), device="cuda")
        engine.mv_g4(ty, w, x, out, m=m, slots=slots, share=share, sel=sel, swiglu=swiglu, ws=ws)
        outs.append(out)
    torch.cuda.synchronize()
    assert torch.isfinite(outs[0]).all() and all(torch.equal(o, outs[0]) for o in outs[1:])
