"""8-bit blocks in 64 bits: codes and scales of rows and matrices, and their products, by the definition in include/kge.h."""
import math

import torch

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3 = torch.float8_e4m3fn
LEAST = 2.0 ** -126


def half_step(dt):
    return torch.finfo(dt).eps / 2


def nearest(v):
    """Numbers of at most 448 in magnitude -> the nearest of e4m3, ties to even."""
    step = torch.exp2(torch.clamp(torch.frexp(v.abs()).exponent - 1, min=-6).double() - 3)
    return torch.round(v / step) * step


def quantise(x, rows):
    """[N, K] -> codes as numbers [N, K] and scales [ceil(N / rows), ceil(K / 128)], in 64 bits; blocks of `rows` x 128."""
    x = x.double()
    N, K = x.shape
    code, scale = torch.zeros_like(x), torch.empty(-(-N // rows), -(-K // 128), dtype=torch.float64)
    for k in range(0, K, 128):
        part = torch.nn.functional.pad(x[:, k:k + 128], (0, 0, 0, -N % rows)).unflatten(0, (-1, rows))
        m = part.abs().amax((1, 2), keepdim=True)                          # (NaN where one is)
        fine = torch.isfinite(m)
        c = nearest(torch.where(fine, torch.where(m >= 448 * LEAST, 448 * part / m, part / LEAST), 0.0))
        code[:, k:k + 128] = c.flatten(0, 1)[:N]
        scale[:, k // 128] = torch.where(fine, torch.clamp(m / 448, min=LEAST), math.nan)[:, 0, 0]
    return code, scale


def numbers(code, scale, rows):
    N, K = code.shape
    return code.double() * scale.double().repeat_interleave(rows, 0)[:N].repeat_interleave(128, 1)[:, :K]


def silu_gate(z):
    g, u = z.chunk(2, -1)
    return g * torch.sigmoid(g) * u
