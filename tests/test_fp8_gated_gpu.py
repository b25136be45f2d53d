"""Gated pairs whose sums are known to the last bit: what silu makes of every gate, and the codes of numbers of 24 bits next to half a step.

Tolerance.  h = g u / (1 + p^2), times p^2 below zero, p = e^(-|g| / 2): a power of two by the unit is off by 2^-22.5 and rounded once, 2^-24, and counts twice
(2 / (1 + p^2)); the sum is rounded, its reciprocal off by 2^-23, four products are rounded: 2^-21.5 + 2^-23 + 2^-24 + 2^-23 + 2^-22 = 8.7e-7, less than 2^-20.  A scale is
rounded once, 2^-24 more.
"""
import math

import pytest
import torch

import fp8_oracle as fo
from test_fp8_gpu import L, call, workspace  # noqa: F401

pytestmark = pytest.mark.gpu
FORMS = [("dense", 3), ("dense", 100), ("dense", 128), ("dense", 300), ("groups", 40), ("groups", 300)]      # shares over a cluster, whole tiles, pairs; by group


def gated_pair(kge, L, form, x, xs, w, ws, T, f):
    """[gate | up] codes w [2 f, K] and scales ws for T rows, all of them the same: codes [T, f] and scales [T, f / 128]."""
    K = x.shape[-1]
    codes, scales, work = torch.full((T, f), 0x55, dtype=torch.uint8, device="cuda"), torch.full((f // 128, T), 9.0, device="cuda"), workspace(L, T)
    args = codes, scales, T, x.expand(T, K).contiguous().cuda(), xs[:, None].expand(-1, T).contiguous().cuda(), T
    if form == "dense":
        call(kge, "kge_gemm_fp8_silu_gate", *args, w.cuda(), ws.cuda(), T, f, K, work, work.numel())
    else:
        off = torch.tensor([0, T // 3, T // 3, T], dtype=torch.int32, device="cuda")
        call(kge, "kge_gemm_fp8_grouped_silu_gate", *args, torch.stack([w] * 3).cuda(), torch.stack([ws] * 3).cuda(), off, 3, T, f, K, work, work.numel())
    torch.cuda.synchronize()
    return codes.cpu().view(fo.E4M3).double(), scales.cpu().t().double()


@pytest.mark.parametrize("form,T", FORMS)
@pytest.mark.parametrize("blocks", [8, 148])
def test_silu_of_every_gate(kge, L, form, T, blocks):
    """One gate and one up in each block of 128, any two fp32 numbers: the block's scale is |h| / 448, for gates from -170 to 88 and ups as large as leave a result."""
    r = torch.Generator().manual_seed(blocks)
    g = torch.empty(blocks).uniform_(-103.0, 88.0, generator=r)
    g[::4] = torch.empty(len(g[::4])).uniform_(-6.0, 6.0, generator=r)
    g[1], g[2], g[3], g[5], g[6] = -87.4, -88.5, -0.0, -20.0, -165.0
    u = 10.0 ** torch.empty(blocks).uniform_(-1.0, 4.0, generator=r)
    u = torch.where(g < -20, u * torch.exp(-g.double() - 30).clamp(max=1e33).float(), u) * (torch.randint(0, 2, (blocks,), generator=r) * 2 - 1)
    u[1], u[2] = 1e3, -4e3
    f, K = 128 * blocks, 272
    x, w = torch.zeros(K), torch.zeros(2, blocks, 128, K)
    x[0] = 1.0
    w[0, :, 17, 0], w[1, :, 17, 0] = 1.0, 1.0
    ws = torch.ones(2 * blocks, 3)
    ws[:blocks, 0], ws[blocks:, 0] = g, u                     # (a scale may be any number: here the sum itself)
    codes, scales = gated_pair(kge, L, form, x.to(fo.E4M3), torch.ones(3), w.view(2 * f, K).to(fo.E4M3), ws, T, f)
    g, u = g.double(), u.double()
    want = torch.clamp((g * torch.sigmoid(g) * u).abs() / 448, min=fo.LEAST)
    assert (want > 2 * fo.LEAST).sum() > blocks - 3
    off = (scales - want).abs() / want
    assert (off <= 2.0 ** -20 + 2.0 ** -24).all(), [(g[i].item(), u[i].item(), off[0, i].item()) for i in off[0].argsort(descending=True)[:5]]
    assert (codes.view(T, blocks, 128)[:, :, [i for i in range(128) if i != 17]] == 0).all()


def digits(u):
    """Whole numbers below 2^24 -> six digits of four bits."""
    return torch.stack([(u >> 4 * b) & 15 for b in range(6)], -1)


def half_steps():
    code = torch.arange(0, 127, dtype=torch.uint8).view(fo.E4M3).double()
    return (code[:-1] + code[1:]) / 2


@pytest.mark.parametrize("form,T", FORMS)
@pytest.mark.parametrize("blocks", [8, 148])
def test_codes_next_to_half_a_step(kge, L, form, T, blocks):
    """The gate is 32 and h = 32 up exactly, up any number of 24 bits, put together of digits with a scale of 16 to the power each: the largest of a block, and for half
    steps t of the codes the two numbers next to t / 448 of it.  Codes and scales bit for bit."""
    r = torch.Generator().manual_seed(blocks)
    up = torch.zeros(blocks, 128, dtype=torch.int64)
    for b in range(blocks):
        m = int(torch.randint(2 ** 23, 2 ** 24, (1,), generator=r)) // (448 if b % 4 == 0 else 1) * (448 if b % 4 == 0 else 1)
        if b % 4 == 1:
            m = m // 7 * 7                                    # (so that some half steps are met exactly)
        t = half_steps()[torch.cat([torch.arange(126 - 40, 126), torch.randint(0, 126 - 40, (23,), generator=r)])]
        low = torch.floor(t * m / 448).long()
        up[b] = torch.cat([torch.tensor([m, m - 1]), low, low + 1])
        up[b] = up[b, torch.randperm(128, generator=r)]
    sign = torch.randint(0, 2, up.shape, generator=r) * 2 - 1
    f, K = 128 * blocks, 7 * 128
    x, w = torch.zeros(K), torch.zeros(2, f, K)
    x[torch.arange(7) * 128 + 5] = 1.0
    w[0, :, 6 * 128 + 5] = 1.0
    w[1][:, torch.arange(6) * 128 + 5] = (digits(up) * sign[..., None]).view(f, 6).float()
    ws = torch.ones(2 * blocks, 7)
    ws[:blocks, 6] = 32.0
    ws[blocks:, :6] = 16.0 ** torch.arange(6)
    codes, scales = gated_pair(kge, L, form, x.to(fo.E4M3), torch.ones(7), w.view(2 * f, K).to(fo.E4M3), ws, T, f)
    code, scale = fo.quantise((32.0 * up * sign).view(1, f), 1)
    assert torch.equal(scales, scale.float().double().expand(T, -1))
    wrong = (codes != code).nonzero()
    assert not len(wrong), (len(wrong), wrong[:5].tolist())
