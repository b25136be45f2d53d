"""8-bit blocks on the GPU: codes and scales bit for bit, products against 64 bits over the same codes, dense, grouped and gated, and all of them
together as a mixture of experts uses them.

Tolerances.  A product's sums are in fp32: over a block of K the matrix unit adds 128 products that are exact (4-bit significands), then K / 128 blocks
are added up.  With A = sum over k of |xs x ws w|, each of at most 128 + K / 128 + 8 additions and scalings is off by a last place of fp32 (2^-23, for a
matrix unit may cut where it should round) of at most A, hence at most n 2^-23 A with n = 136 + K / 128: what a sum is held to.  A 16-bit result
is rounded once more, u |y| with u = eps / 2.  In the 2-norm that rounding alone counts, u / sqrt(3) where significands are spread evenly, held to u.
A gated pair: h = silu(g) u has the derivatives |dh/dg| <= 1.1 |u| and |silu(g)| in them, and e^-g and the quotient are off by 2^-20 (|g| up to 88) of it.
Codes are off by half a step of 8 bits, 2^-4 of the value, or 2^-10 of the scale where it is below the normal range; the scale by as much as the
largest h.
"""
import math

import numpy as np
import pytest
import torch

import fp8_oracle as fo

pytestmark = pytest.mark.gpu
I32 = dict(dtype=torch.int32, device="cuda")


@pytest.fixture(scope="module")
def L(kge):
    kge.require_cuda()
    return kge.lib()


def name(fn, dt):
    return fn + ("_f16" if dt == torch.float16 else "")


def call(kge, fn, *args, stream=None):
    rc = getattr(kge.lib(), fn)(*[a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args], (stream or torch.cuda.current_stream()).cuda_stream)
    kge.check(rc, fn)


def workspace(L, T, fill=0xFF):
    """What the call asks for and no more; only the counters at its head have to be zero."""
    ws = torch.full((max(1024, L.kge_gemm_fp8_workspace_bytes(T)),), fill, dtype=torch.uint8, device="cuda")
    ws[:1024] = 0
    return ws


def rows_of(g, T, K, dt):
    x = torch.randn(T, K, generator=g) * torch.exp(torch.randn(T, 1, generator=g))
    x[:, torch.rand(K, generator=g) < 0.02] *= 30
    return x.to(dt)


def quantised(g, T, K, rows):
    """Codes (e4m3), scales by blocks, and the numbers that they stand for in 64 bits."""
    x = rows_of(g, T, K, torch.bfloat16) if rows == 1 else (torch.randn(T, K, generator=g) * K ** -0.5).to(torch.bfloat16)
    code, scale = fo.quantise(x, rows)
    scale = scale.float()
    return code.to(fo.E4M3), scale, fo.numbers(code, scale, rows)


# ---------------------------------------------------------------------------------------------------------------- quantising

QUANT = [("bf16", 1, 16), ("fp16", 1, 128), ("bf16", 3, 144), ("fp16", 33, 1424), ("bf16", 64, 4096), ("fp16", 200, 272), ("bf16", 7, 14336)]


@pytest.mark.parametrize("dtype,T,K", QUANT)
@pytest.mark.parametrize("form", ["plain", "strided", "gathered"])
def test_rows_are_quantised_bit_for_bit(kge, L, dtype, T, K, form):
    dt, g = fo.DT[dtype], torch.Generator().manual_seed(T + K)
    x = rows_of(g, T, K, dt)
    code, scale = fo.quantise(x, 1)
    stride = T if form == "plain" else T + 5
    codes, scales = torch.full((T + 1, K), 0x55, dtype=torch.uint8, device="cuda"), torch.full((scale.shape[1], stride), 9.0, device="cuda")
    rows, src = None, x.cuda()
    if form == "strided":
        src = torch.full((T, K + 24), 3e4, dtype=dt, device="cuda")
        src[:, :K] = x
    if form == "gathered":
        at = torch.randint(-1, T, (T,), generator=g)
        code, scale = code[at], scale[at]
        code[at < 0], scale[at < 0] = 0.0, fo.LEAST
        rows = at.int().cuda()
    call(kge, name("kge_fp8_quant", dt), codes, scales, stride, src, src.shape[1], rows, T, K)
    torch.cuda.synchronize()
    assert torch.equal(codes[:T].cpu().view(fo.E4M3).double(), code)
    assert torch.equal(scales[:, :T].cpu().t(), scale.float())
    assert (codes[T:] == 0x55).all() and (scales[:, T:] == 9).all()


@pytest.mark.parametrize("dtype,E,N,K", [("bf16", 1, 1, 16), ("fp16", 1, 128, 128), ("bf16", 3, 200, 144), ("fp16", 2, 129, 272), ("bf16", 1, 640, 1424), ("bf16", 5, 64, 48)])
def test_weights_are_quantised_bit_for_bit(kge, L, dtype, E, N, K):
    dt, g = fo.DT[dtype], torch.Generator().manual_seed(N + K)
    w = torch.randn(E, N, K, generator=g).to(dt)
    want = [fo.quantise(m, 128) for m in w]
    codes, scales = torch.full((E * N + 1, K), 0x55, dtype=torch.uint8, device="cuda"), torch.full((E * want[0][1].numel() + 1,), 9.0, device="cuda")
    call(kge, name("kge_fp8_quant_weight", dt), codes, scales, w.cuda(), E, N, K)
    torch.cuda.synchronize()
    assert torch.equal(codes[:-1].cpu().view(fo.E4M3).double(), torch.cat([c for c, _ in want]))
    assert torch.equal(scales[:-1].cpu(), torch.cat([s.flatten() for _, s in want]).float())
    assert (codes[-1] == 0x55).all() and scales[-1] == 9


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_every_tie_and_every_magnitude(kge, L, dtype):
    """For largest magnitudes of every significand, numbers of every significand and 20 exponents below it: halves of a step go to the even code."""
    dt = fo.DT[dtype]
    n = 1 << (7 if dt == torch.bfloat16 else 10)
    sig = torch.arange(n, 2 * n).double() / n
    tops = sig[:: n // 128]
    rows = []
    for d in range(21):
        x = (sig * 2.0 ** -d)[:: 1 if n == 128 else 5]
        rows.append(torch.nn.functional.pad(x, (0, -len(x) % 127)).view(-1, 127))
    body = torch.cat(rows)
    x = torch.cat([torch.cat([torch.full((len(body), 1), t.item()), torch.minimum(body, t)], 1) for t in tops])
    x = (x * (torch.arange(128) % 2 * 2 - 1)).to(dt)
    code, scale = fo.quantise(x, 1)
    codes, scales = torch.zeros(x.shape, dtype=torch.uint8, device="cuda"), torch.zeros(1, len(x), device="cuda")
    call(kge, name("kge_fp8_quant", dt), codes, scales, len(x), x.cuda(), 128, None, len(x), 128)
    torch.cuda.synchronize()
    assert torch.equal(codes.cpu().view(fo.E4M3).double(), code) and torch.equal(scales[0].cpu(), scale[:, 0].float())


SPECIAL = {"zeros": 0.0, "inf": math.inf, "minus inf": -math.inf, "nan": math.nan, "largest": None, "tiny": 1e-7, "least": 6e-8}


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kind", sorted(SPECIAL) + ["denormal bf16"])
def test_blocks_of_special_numbers(kge, L, dtype, kind):
    """An infinity or NaN makes its block's scale NaN and its codes zero, and no other block's; zeros have the least scale."""
    dt = fo.DT[dtype]
    if kind == "denormal bf16":
        if dtype == "fp16":
            pytest.skip("float16 has nothing that small")
        v = 3e-39
    else:
        v = torch.finfo(dt).max if SPECIAL[kind] is None else SPECIAL[kind]
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 400, generator=g).to(dt)
    if math.isfinite(v) and kind != "largest":
        x[2, 128:256] = v
    else:
        x[2, 200] = v
        x[4, 399] = -v
    code, scale = fo.quantise(x, 1)
    codes, scales = torch.zeros(5, 400, dtype=torch.uint8, device="cuda"), torch.zeros(4, 5, device="cuda")
    call(kge, name("kge_fp8_quant", dt), codes, scales, 5, x.cuda(), 400, None, 5, 400)
    wcode, wscale = fo.quantise(x, 128)
    wcodes, wscales = torch.zeros(5, 400, dtype=torch.uint8, device="cuda"), torch.zeros(4, device="cuda")
    call(kge, name("kge_fp8_quant_weight", dt), wcodes, wscales, x.cuda(), 1, 5, 400)
    torch.cuda.synchronize()
    for got, s, want, ws in ((codes, scales.t(), code, scale), (wcodes, wscales[None], wcode, wscale)):
        assert torch.equal(got.cpu().view(fo.E4M3).double(), want)
        assert torch.equal(torch.nan_to_num(s.cpu(), nan=-1.0), torch.nan_to_num(ws.float(), nan=-1.0))


# ------------------------------------------------------------------------------------------------------------------ products

def held(y, z, a, K, u):
    """A product against 64 bits: z the sums, a the sums of magnitudes."""
    y = y.double()
    n = (136 + K / 128) * 2.0 ** -23
    assert ((y - z).abs() <= n * a + u * (z.abs() + n * a) + 1e-30).all(), ((y - z).abs() - n * a - u * z.abs()).max()
    if z.numel() >= 512:
        assert (y - z).norm() <= u * z.norm()


def held_gated(codes, scales, z, a, K):
    """Codes [T, f] and scales [T, f / 128] of a gated pair against 64 bits: z, a as for held, [T, 2 f]."""
    h = fo.silu_gate(z)
    e = (136 + K / 128) * 2.0 ** -23 * a
    g, u = z.chunk(2, -1)
    eg, eu = e.chunk(2, -1)
    off = (1.1 * (u.abs() + eu) * eg + (g * torch.sigmoid(g)).abs() * eu) + 2.0 ** -20 * h.abs() + 1e-30
    block = h.unflatten(1, (-1, 128))
    top = block.abs().amax(-1)
    slack = off.unflatten(1, (-1, 128)).amax(-1)
    want = torch.clamp(top / 448, min=fo.LEAST)
    assert ((scales.double() - want).abs() <= slack / 448 + 2.0 ** -23 * want).all()
    s = scales.double().repeat_interleave(128, 1)
    got = codes.double() * s
    assert ((got - h).abs() <= 2.0 ** -4 * h.abs() + 2.0 ** -10 * s + 1.1 * off + slack.repeat_interleave(128, 1) * (h.abs() / top.repeat_interleave(128, 1).clamp(min=1e-30))).all()


GEMM = [  # T, N, K
    (1, 1, 16), (1, 128, 128), (1, 4096, 512), (2, 8, 144), (3, 129, 272), (16, 256, 1024), (17, 1000, 2064), (31, 640, 4096), (32, 96, 128), (33, 2504, 384),
    (64, 6144, 1024), (65, 136, 14336), (100, 3000, 640), (127, 520, 1424), (128, 1024, 1024), (129, 384, 528), (200, 1031, 1296), (256, 512, 2048), (257, 264, 400),
    (300, 1000, 272), (511, 640, 144), (512, 2048, 1024), (700, 1288, 2064), (1339, 777, 656)]


@pytest.mark.parametrize("T,N,K", GEMM)
@pytest.mark.parametrize("dtype,bias", [("bf16", False), ("fp16", True)])
def test_product(kge, L, T, N, K, dtype, bias):
    dt, g = fo.DT[dtype], torch.Generator().manual_seed(T + N + K)
    x, xs, xn = quantised(g, T, K, 1)
    w, ws, wn = quantised(g, N, K, 128)
    b = torch.randn(N, generator=g).to(dt) if bias else None
    y = torch.full((T + 1, N), 7.0, dtype=dt, device="cuda")
    work = workspace(L, T)
    args = x.cuda(), xs.t().contiguous().cuda(), T, w.cuda(), ws.cuda(), b.cuda() if bias else None, T, N, K, work, work.numel()
    call(kge, name("kge_gemm_fp8", dt), y, *args)
    torch.cuda.synchronize()
    z, a = xn @ wn.t(), xn.abs() @ wn.abs().t()
    if bias:
        z, a = z + b.double(), a + b.double().abs()
    held(y[:T].cpu(), z, a, K, fo.half_step(dt))
    assert (y[T] == 7).all() and (work[:1024] == 0).all()
    again = torch.zeros_like(y)
    call(kge, name("kge_gemm_fp8", dt), again, *args)
    torch.cuda.synchronize()
    assert torch.equal(again[:T], y[:T])                                    # the same bits each time


GATED = [(1, 128, 128), (1, 1024, 528), (5, 256, 144), (33, 384, 1040), (64, 2048, 1024), (96, 640, 2064), (128, 128, 4096), (130, 512, 272), (256, 256, 640), (257, 384, 1424),
         (600, 896, 400)]


@pytest.mark.parametrize("T,f,K", GATED)
def test_gated_pair(kge, L, T, f, K):
    g = torch.Generator().manual_seed(T + f + K)
    x, xs, xn = quantised(g, T, K, 1)
    w, ws, wn = quantised(g, 2 * f, K, 128)
    codes, scales = torch.full((T + 1, f), 0x55, dtype=torch.uint8, device="cuda"), torch.full((f // 128, T + 3), 9.0, device="cuda")
    work = workspace(L, T)
    xd = torch.full((xs.shape[1], T + 2), math.nan, device="cuda")                        # a stride of its own
    xd[:, :T] = xs.t()
    call(kge, "kge_gemm_fp8_silu_gate", codes, scales, T + 3, x.cuda(), xd, T + 2, w.cuda(), ws.cuda(), T, f, K, work, work.numel())
    torch.cuda.synchronize()
    held_gated(codes[:T].cpu().view(fo.E4M3), scales[:, :T].cpu().t(), xn @ wn.t(), xn.abs() @ wn.abs().t(), K)
    assert (codes[T] == 0x55).all() and (scales[:, T:] == 9).all() and (work[:1024] == 0).all()


GROUPS = [  # rows of each group, N, K
    ([1], 64, 128), ([0, 0, 3], 200, 272), ([5, 0, 1, 0, 0, 40], 136, 528), ([128, 127, 129], 300, 400), ([0] * 30 + [7], 128, 144), ([1] * 70, 264, 256),
    ([300, 2, 0, 33], 512, 1040), ([0, 0, 0], 128, 128), ([3] * 8, 1536, 1024), ([260, 255, 0, 513, 700], 392, 272), ([900], 640, 528), ([2, 1500, 1, 600], 256, 656),
    ([4] * 300, 64, 48), ([31, 32, 33, 64, 65, 96, 97], 768, 144)]


@pytest.mark.parametrize("sizes,N,K", GROUPS, ids=lambda v: str(v) if isinstance(v, int) else "x".join(map(str, v))[:24])
@pytest.mark.parametrize("form", ["bf16", "fp16", "gated"])
@pytest.mark.parametrize("first,behind", [(0, 0), (3, 9)])
def test_grouped(kge, L, sizes, N, K, form, first, behind):
    """Rows before the first group and behind the last one are left as they were."""
    E, T = len(sizes), first + sum(sizes) + behind
    if T == 0:
        T = behind = 2
    off = [first + s for s in np.concatenate([[0], np.cumsum(sizes)]).tolist()]
    g = torch.Generator().manual_seed(T + N + K)
    gated = form == "gated"
    N = -(-N // 128) * 256 if gated else N                                  # rows of a matrix
    x, xs, xn = quantised(g, T, K, 1)
    parts = [quantised(g, N, K, 128) for _ in range(min(E, 8))]             # (matrices repeat: groups still have places of their own)
    w, ws, wn = ([parts[e % len(parts)][i] for e in range(E)] for i in range(3))
    wd, wsd = torch.stack(w).cuda(), torch.stack(ws).cuda()
    work, offsets = workspace(L, T), torch.tensor(off, **I32)
    xsd = xs.t().contiguous().cuda()
    if gated:
        f = N // 2
        codes, scales = torch.full((T, f), 0x55, dtype=torch.uint8, device="cuda"), torch.full((f // 128, T), 9.0, device="cuda")
        call(kge, "kge_gemm_fp8_grouped_silu_gate", codes, scales, T, x.cuda(), xsd, T, wd, wsd, offsets, E, T, f, K, work, work.numel())
    else:
        dt = fo.DT[form]
        y = torch.full((T, N), 7.0, dtype=dt, device="cuda")
        call(kge, name("kge_gemm_fp8_grouped", dt), y, x.cuda(), xsd, T, wd, wsd, offsets, E, T, N, K, work, work.numel())
    torch.cuda.synchronize()
    z, a = torch.zeros(T, N, dtype=torch.float64), torch.zeros(T, N, dtype=torch.float64)
    for e in range(E):
        r = slice(off[e], off[e + 1])
        z[r], a[r] = xn[r] @ wn[e].t(), xn[r].abs() @ wn[e].abs().t()
    r, other = slice(off[0], off[-1]), torch.tensor([i for i in range(T) if not off[0] <= i < off[-1]], dtype=torch.long)
    if gated:
        if off[-1] > off[0]:
            held_gated(codes[r].cpu().view(fo.E4M3), scales[:, r].cpu().t(), z[r], a[r], K)
        assert (codes.cpu()[other] == 0x55).all() and (scales.cpu()[:, other] == 9).all()
    else:
        if off[-1] > off[0]:
            held(y[r].cpu(), z[r], a[r], K, fo.half_step(dt))
        assert (y.cpu()[other] == 7).all()
    assert (work[:1024] == 0).all()


@pytest.mark.parametrize("off", [[0, 5, 3, 9], [-4, 2, 2, 70], [9, 3, 1, 0], [50, 60, 70, 80], [2 ** 31 - 1, -2 ** 31, 0, 12]])
def test_offsets_that_are_none_stay_within_the_rows(kge, L, off):
    """Offsets that fall or lie outside of the rows: nothing outside of y is written."""
    T, N, K, g = 20, 136, 144, torch.Generator().manual_seed(0)
    x, xs, _ = quantised(g, T, K, 1)
    w, ws, _ = quantised(g, N, K, 128)
    whole = torch.full((T + 200, N), 7.0, dtype=torch.bfloat16, device="cuda")
    work = workspace(L, T)
    call(kge, "kge_gemm_fp8_grouped", whole[100:], x.cuda(), xs.t().contiguous().cuda(), T, torch.stack([w] * 3).cuda(), torch.stack([ws] * 3).cuda(), torch.tensor(off, **I32), 3, T, N, K,
         work, work.numel())
    torch.cuda.synchronize()
    assert (whole[:100] == 7).all() and (whole[100 + T:] == 7).all() and (work[:1024] == 0).all()
