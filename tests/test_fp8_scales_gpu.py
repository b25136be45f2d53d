"""Products whose two scales multiply to numbers next to the ends of fp32.

Tolerance, beside what any product is held to (n 2^-23 of the sum of magnitudes, n = 136 + K / 128, and half a step of the result): a factor xs ws below 2^-126 is rounded
to 2^-150, times the block's sum of codes; each addition may be rounded to 2^-150 too, and the result to half of bfloat16's smallest step, 2^-134.
"""
import math

import pytest
import torch

import fp8_oracle as fo
from test_fp8_gpu import L, call, quantised, workspace  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,N,K", [(10, 400, 256), (10, 3000, 1040), (100, 1031, 528), (700, 1288, 400)])      # shares over a cluster, whole tiles, unaligned rows, pairs
def test_products_of_scales_at_the_ends(kge, L, T, N, K):
    g = torch.Generator().manual_seed(T + N)
    x, xs, _ = quantised(g, T, K, 1)
    w, ws, _ = quantised(g, N, K, 128)                         # (their scales lie about 2^-11)
    tiny, big, beyond, none = [0, 1, 2, T - 1], 3, 4, 5
    xs[0], xs[1], xs[2], xs[T - 1] = 2.0 ** -126, 1.5 * 2.0 ** -124, 2.0 ** -120, 1.1 * 2.0 ** -126
    xs[big], xs[beyond], xs[none] = 2.0 ** 110, 2.0 ** 127, 0.0
    ws[0, 0] = 2.0                                             # with row `beyond` it is beyond the end, in the first 128 columns
    y = torch.full((T, N), 7.0, dtype=torch.bfloat16, device="cuda")
    work = workspace(L, T)
    call(kge, "kge_gemm_fp8", y, x.cuda(), xs.t().contiguous().cuda(), T, w.cuda(), ws.cuda(), None, T, N, K, work, work.numel())
    y = y.cpu().double()
    xc, wc = x.double(), w.double()
    xn, wn = fo.numbers(xc, xs, 1), fo.numbers(wc, ws, 128)
    z, a, codes = xn @ wn.t(), xn.abs() @ wn.abs().t(), xc.abs() @ wc.abs().t()
    n = (136 + K / 128) * 2.0 ** -23
    off = n * a + fo.half_step(torch.bfloat16) * (z.abs() + n * a) + 2.0 ** -150 * (codes + K / 128) + 2.0 ** -134
    rows = [t for t in range(T) if t != beyond]
    most = torch.finfo(torch.bfloat16).max
    beyond16 = (y == z.sign() * math.inf) & (z.abs() + off > most)      # (what bfloat16 does not hold)
    assert (((y - z).abs() <= off) | beyond16)[rows].all() and beyond16[rows].any()
    assert (z[tiny].abs() > 8 * off[tiny]).double().mean() > 0.9, "the test would see nothing"
    assert (ws[1:].max() * 2.0 ** -126) < 2.0 ** -130 and not y[beyond, :128].isfinite().any() and (y[none] == 0).all()
