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

QUANT = [("bf16", 1, 16), ("fp16", 1, 128), ("bf16", 3, 144), ("fp16", 33, 1424), ("bf16", 64, 4096), ("fp16", 200, 272), ("bf16", 7, 14336), ("bf16", 9700, 528), ("fp16", 4800, 1040)]


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


TILES = [  # T, N, K: whole tiles of 256 columns, one and several a CTA; tiles of 128 columns cut along K over 2 to 8 CTAs; pairs, whole and ragged
    (5, 19000, 272), (3, 40000, 144), (130, 19000, 144), (40, 30000, 1424), (1, 6016, 2048), (64, 4096, 528), (9, 2048, 1040), (33, 384, 2064), (97, 256, 4096), (128, 128, 4112),
    (65, 1536, 1296), (120, 9500, 400), (1030, 4104, 272), (2050, 2056, 528), (3000, 600, 144), (520, 8200, 400)]


@pytest.mark.parametrize("T,N,K", TILES)
def test_product_in_every_kind_of_tile(kge, L, T, N, K):
    g = torch.Generator().manual_seed(T + N)
    x, xs, xn = quantised(g, T, K, 1)
    w, ws, wn = quantised(g, N, K, 128)
    y = torch.full((T + 1, N), 7.0, dtype=torch.bfloat16, device="cuda")
    work = workspace(L, T)
    call(kge, "kge_gemm_fp8", y, x.cuda(), xs.t().contiguous().cuda(), T, w.cuda(), ws.cuda(), None, T, N, K, work, work.numel())
    xn, wn = xn.cuda(), wn.cuda()
    z, a = (xn @ wn.t()).cpu(), (xn.abs() @ wn.abs().t()).cpu()
    held(y[:T].cpu(), z, a, K, fo.half_step(torch.bfloat16))
    assert (y[T] == 7).all() and (work[:1024] == 0).all()


@pytest.mark.parametrize("K", [128, 400])
def test_every_number_of_rows_and_columns(kge, L, K):
    """1 to 140 rows of 72 columns and 1 to 140 columns of 3 rows: sentinels around the result stay."""
    g = torch.Generator().manual_seed(K)
    x, xs, xn = quantised(g, 140, K, 1)
    w, ws, wn = quantised(g, 140, K, 128)
    xd, xsd, wd, wsd = x.cuda(), xs.t().contiguous().cuda(), w.cuda(), ws.cuda()
    z, a = xn @ wn.t(), xn.abs() @ wn.abs().t()
    work = workspace(L, 140)
    for T, N in [(t, 72) for t in range(1, 141)] + [(3, n) for n in range(1, 141)]:
        y = torch.full((T * N + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
        call(kge, "kge_gemm_fp8", y[32:], xd, xsd, 140, wd, wsd, None, T, N, K, work, work.numel())
        got = y.cpu()
        assert (got[:32] == 7).all() and (got[32 + T * N:] == 7).all(), (T, N)
        held(got[32:32 + T * N].view(T, N), z[:T, :N], a[:T, :N], K, fo.half_step(torch.bfloat16))


def test_what_is_no_number_stays_in_its_row_or_columns(kge, L):
    """A row's NaN scale, NaN code or infinite scale makes its own results NaN or infinite; a block of weights its 128 columns; nothing else changes."""
    T, N, K, g = 40, 400, 528, torch.Generator().manual_seed(5)
    x, xs, _ = quantised(g, T, K, 1)
    w, ws, _ = quantised(g, N, K, 128)
    work = workspace(L, T)

    def run(x, xs, w, ws):
        y = torch.zeros(T, N, dtype=torch.bfloat16, device="cuda")
        call(kge, "kge_gemm_fp8", y, x.cuda(), xs.t().contiguous().cuda(), T, w.cuda(), ws.cuda(), None, T, N, K, work, work.numel())
        return y.cpu()
    want = run(x, xs, w, ws)
    xs2, ws2, x2 = xs.clone(), ws.clone(), x.clone()
    xs2[3, 1], xs2[7, 0], ws2[1, 2] = math.nan, math.inf, math.nan
    x2.view(torch.uint8)[33, 17] = 0x7f
    got = run(x2, xs2, w, ws2)
    bad = torch.zeros(T, N, dtype=torch.bool)
    bad[[3, 33]], bad[:, 128:256] = True, True
    assert got[bad].isnan().all() and not got[7].isfinite().any()
    bad[7] = True
    assert torch.equal(got[~bad], want[~bad])
    # and through the gated pair: the row's blocks are NaN, with codes of zero
    wg, wgs, _ = quantised(g, 512, K, 128)
    codes, scales = torch.full((T, 256), 0x55, dtype=torch.uint8, device="cuda"), torch.zeros(2, T, device="cuda")
    call(kge, "kge_gemm_fp8_silu_gate", codes, scales, T, x2.cuda(), xs2.t().contiguous().cuda(), T, wg.cuda(), wgs.cuda(), T, 256, K, work, work.numel())
    rows = torch.zeros(T, dtype=torch.bool)
    rows[[3, 7, 33]] = True
    assert scales.cpu()[:, rows].isnan().all() and (codes.cpu()[rows] == 0).all() and scales.cpu()[:, ~rows].isfinite().all()


def test_zero_and_extreme_scales(kge, L):
    """Rows of zeros, scales of 2^-126 and 2^120: sums neither vanish nor overflow before they have to."""
    T, N, K, g = 8, 136, 256, torch.Generator().manual_seed(6)
    x, xs, _ = quantised(g, T, K, 1)
    w, ws, _ = quantised(g, N, K, 128)
    xs[0], xs[1], xs[2] = 2.0 ** -126, 2.0 ** 100, 0.0
    x.view(torch.uint8)[3] = 0
    ws = ws * 2.0 ** 10
    y = torch.zeros(T, N, dtype=torch.bfloat16, device="cuda")
    work = workspace(L, T)
    call(kge, "kge_gemm_fp8", y, x.cuda(), xs.t().contiguous().cuda(), T, w.cuda(), ws.cuda(), None, T, N, K, work, work.numel())
    xn, wn = fo.numbers(x.double(), xs, 1), fo.numbers(w.double(), ws, 128)
    held(y.cpu(), xn @ wn.t(), xn.abs() @ wn.abs().t() + 2.0 ** -126 * 448 * 448 * K, K, fo.half_step(torch.bfloat16))
    assert (y[2:4] == 0).all()


# ------------------------------------------------------------------------------------------------- as they are used together

def experts64(x, wg, wd, chosen, share):
    """A mixture in 64 bits over the quantised numbers, and what the result is held to (see below)."""
    out, mag = torch.zeros(x.shape[0], wd[0].shape[0], dtype=torch.float64), torch.zeros(x.shape[0], dtype=torch.float64)
    for t in range(x.shape[0]):
        for k, e in enumerate(chosen[t].tolist()):
            h = fo.silu_gate((x[t] @ wg[e].t())[None])[0]
            out[t] += share[t, k] * (wd[e] @ h)
            mag[t] += share[t, k] * wd[e].norm(dim=1).max() * h.norm()
    return out, mag


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tokens,E,top,d,f", [(1, 4, 2, 256, 128), (9, 16, 4, 512, 256), (200, 8, 2, 384, 256), (900, 4, 2, 256, 384)])
def test_a_mixture_of_experts(kge, L, dtype, tokens, E, top, d, f):
    """Weights quantised, tokens gathered by expert and quantised, gate and up, down: one stream, nothing waits for the host.  Against the experts over the
    numbers that the codes stand for.  Between the products h has 8 bits: each number off by 2^-4 of it at most, in the mean square 2^-4 / sqrt(3) of it and
    2^-5 where significands are spread; a result, a sum of f of them, is off by the norm of the weights' row times that of h times 2^-5 / sqrt(3) or so in
    the mean square, held to 2^-4 of the two norms (codes below the normal range, 2^-10 of a block's scale, are less)."""
    dt, g = fo.DT[dtype], torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, d, generator=g).to(dt)
    wg, wd = (torch.randn(E, 2 * f, d, generator=g) * d ** -0.5).to(dt), (torch.randn(E, d, f, generator=g) * f ** -0.5).to(dt)
    chosen = torch.stack([torch.randperm(E, generator=g)[:top] for _ in range(tokens)])
    share = torch.softmax(torch.randn(tokens, top, generator=g), -1).double()
    pair = chosen.flatten().sort(stable=True)
    T = tokens * top
    rows, off = (pair.indices // top).int().cuda(), torch.cat([torch.zeros(1, dtype=torch.long), torch.bincount(pair.values, minlength=E).cumsum(0)]).int().cuda()
    u8, f32 = dict(dtype=torch.uint8, device="cuda"), dict(device="cuda")
    cg, sg, cd, sd = torch.empty(E, 2 * f, d, **u8), torch.empty(E, -(-2 * f // 128), -(-d // 128), **f32), torch.empty(E, d, f, **u8), torch.empty(E, -(-d // 128), f // 128, **f32)
    cx, sx, ch, sh = torch.empty(T, d, **u8), torch.empty(-(-d // 128), T, **f32), torch.empty(T, f, **u8), torch.empty(f // 128, T, **f32)
    y, work = torch.empty(T, d, dtype=dt, device="cuda"), workspace(L, T)
    xd, wgd, wdd = x.cuda(), wg.cuda(), wd.cuda()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    call(kge, name("kge_fp8_quant_weight", dt), cg, sg, wgd, E, 2 * f, d, stream=st)
    call(kge, name("kge_fp8_quant_weight", dt), cd, sd, wdd, E, d, f, stream=st)
    call(kge, name("kge_fp8_quant", dt), cx, sx, T, xd, d, rows, T, d, stream=st)
    call(kge, "kge_gemm_fp8_grouped_silu_gate", ch, sh, T, cx, sx, T, cg, sg, off, E, T, f, d, work, work.numel(), stream=st)
    call(kge, name("kge_gemm_fp8_grouped", dt), y, ch, sh, T, cd, sd, off, E, T, d, f, work, work.numel(), stream=st)
    st.synchronize()
    pairs = torch.empty(T, d, dtype=torch.float64)
    pairs[pair.indices] = y.double().cpu()
    got = (pairs.view(tokens, top, d) * share[..., None]).sum(1)
    num = lambda c, s, r: fo.numbers(c.cpu().view(fo.E4M3).double(), s.cpu(), r)
    xn, xscale = fo.quantise(x, 1)
    want, mag = experts64(fo.numbers(xn, xscale.float(), 1), [num(cg[e], sg[e], 128) for e in range(E)], [num(cd[e], sd[e], 128) for e in range(E)], chosen, share)
    assert ((got - want).abs() <= 2.0 ** -4 * mag[:, None]).all()
    assert (got - want).norm() <= (2.0 ** -4 / math.sqrt(3) + fo.half_step(dt)) * want.norm()


def test_a_captured_step_over_changing_groups(kge, L):
    """Two graphs that share a workspace, replayed in turn with other rows, offsets and numbers of rows: each gives what calls of the time give."""
    E, T, d, f, g = 6, 70, 256, 128, torch.Generator().manual_seed(11)
    w, ws, _ = quantised(g, E * 2 * f, d, 128)
    w2, ws2, _ = quantised(g, E * d, f, 128)
    w, ws, w2, ws2 = w.cuda(), ws.cuda(), w2.cuda(), ws2.cuda()
    x, off = torch.zeros(T, d, dtype=torch.bfloat16, device="cuda"), torch.zeros(E + 1, **I32)
    u8, f32 = dict(dtype=torch.uint8, device="cuda"), dict(device="cuda")
    work = workspace(L, T)

    def buffers():
        return (torch.zeros(T, d, **u8), torch.zeros(2, T, **f32), torch.zeros(T, f, **u8), torch.zeros(1, T, **f32), torch.zeros(T, d, dtype=torch.bfloat16, device="cuda"))

    def step(b):
        cx, sx, ch, sh, y = b
        call(kge, "kge_fp8_quant", cx, sx, T, x, d, None, T, d)
        call(kge, "kge_gemm_fp8_grouped_silu_gate", ch, sh, T, cx, sx, T, w, ws, off, E, T, f, d, work, work.numel())
        call(kge, "kge_gemm_fp8_grouped", y, ch, sh, T, w2, ws2, off, E, T, d, f, work, work.numel())

    def dense(b):
        cx, sx, ch, sh, y = b
        call(kge, "kge_gemm_fp8_silu_gate", ch, sh, T, cx, sx, T, w, ws, T, f, d, work, work.numel())
        call(kge, "kge_gemm_fp8", y, ch, sh, T, w2, ws2, None, T, d, f, work, work.numel())
    eager, a, b = buffers(), buffers(), buffers()
    step(eager), dense(eager)
    torch.cuda.synchronize()
    graphs = []
    for fn, buf in ((step, a), (dense, b)):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            fn(buf)
        graphs.append(gr)
    for turn in range(6):
        x.copy_(torch.randn(T, d, generator=g) * 10 ** (turn - 2))
        sizes = torch.randint(0, 12, (E,), generator=g)
        sizes[turn] = 0
        off.copy_(torch.cat([torch.zeros(1, dtype=torch.long), sizes.cumsum(0)]))
        for t in (*eager, *a, *b):
            t.zero_()
        b[0].copy_(a[0])
        graphs[0].replay()
        step(eager)
        torch.cuda.synchronize()
        for s, t in zip(a, eager):
            assert torch.equal(s.view(torch.uint8), t.view(torch.uint8)), turn
        b[0].copy_(a[0]), b[1].copy_(a[1])
        graphs[1].replay()
        eager2 = [a[0], a[1], *(torch.zeros_like(t) for t in a[2:])]
        dense(eager2)
        torch.cuda.synchronize()
        for s, t in zip(b, eager2):
            assert torch.equal(s.view(torch.uint8), t.view(torch.uint8)), turn
    assert (work[:1024] == 0).all()


def test_two_streams_at_once(kge, L):
    """Calls on two streams with a workspace each, many times: the bits that each gives alone."""
    g = torch.Generator().manual_seed(12)
    jobs = []
    for T, N, K in ((3, 640, 2064), (300, 776, 528)):
        x, xs, _ = quantised(g, T, K, 1)
        w, ws, _ = quantised(g, N, K, 128)
        y = torch.zeros(T, N, dtype=torch.bfloat16, device="cuda")
        work = workspace(L, T)
        off = torch.tensor([0, T // 3, T // 3, T], **I32)
        args = x.cuda(), xs.t().contiguous().cuda(), T, torch.stack([w] * 3).cuda(), torch.stack([ws] * 3).cuda(), off, 3, T, N, K, work, work.numel()
        call(kge, "kge_gemm_fp8_grouped", y, *args)
        torch.cuda.synchronize()
        jobs.append((torch.cuda.Stream(), args, y.clone(), [torch.zeros_like(y) for _ in range(20)]))
    for i in range(20):
        for st, args, _, ys in jobs:
            call(kge, "kge_gemm_fp8_grouped", ys[i], *args, stream=st)
    torch.cuda.synchronize()
    for _, _, want, ys in jobs:
        assert all(torch.equal(y, want) for y in ys)


def test_a_slice_of_a_batch(kge, L):
    """Rows t0 .. of a quantised batch: codes and scales from there on, with the batch's stride."""
    T, N, K, g = 50, 200, 272, torch.Generator().manual_seed(13)
    x, xs, _ = quantised(g, T, K, 1)
    w, ws, _ = quantised(g, N, K, 128)
    xd, xsd, wd, wsd, work = x.cuda(), xs.t().contiguous().cuda(), w.cuda(), ws.cuda(), workspace(L, T)
    whole = torch.zeros(T, N, dtype=torch.bfloat16, device="cuda")
    call(kge, "kge_gemm_fp8", whole, xd, xsd, T, wd, wsd, None, T, N, K, work, work.numel())
    for t0, n in ((1, 3), (17, 33), (49, 1)):
        y = torch.zeros(n, N, dtype=torch.bfloat16, device="cuda")
        call(kge, "kge_gemm_fp8", y, xd[t0:], xsd.flatten()[t0:], T, wd, wsd, None, n, N, K, work, work.numel())
        assert torch.equal(y, whole[t0:t0 + n])


def test_more_than_32_bits_of_elements(kge, L):
    """A result of 2^31 numbers and more, weights of 2^31 bytes and more, rows beyond 2^31 numbers: the last of each are right."""
    g = torch.Generator().manual_seed(14)
    T, N, K = 66000, 33024, 128
    x, xs, xn = quantised(g, 512, K, 1)
    w, ws, wn = quantised(g, 256, K, 128)
    xd, xsd = x.view(torch.uint8).cuda().repeat(T // 512 + 1, 1)[:T].contiguous(), xs.t().contiguous().cuda().repeat(1, T // 512 + 1)[:, :T].contiguous()
    wd, wsd = w.view(torch.uint8).cuda().repeat(N // 256, 1).contiguous(), ws.cuda().repeat(N // 256, 1).contiguous()
    y, work = torch.zeros(T, N, dtype=torch.bfloat16, device="cuda"), workspace(L, T)
    call(kge, "kge_gemm_fp8", y, xd, xsd, T, wd, wsd, None, T, N, K, work, work.numel())
    z, a = xn @ wn.t(), xn.abs() @ wn.abs().t()
    at = torch.arange(T - 300, T) % 512
    for n in (0, N - 256):
        held(y[T - 300:, n:n + 256].cpu(), z[at], a[at], K, fo.half_step(torch.bfloat16))
    del y, wd
    E = 2                                                    # the second group's matrix begins behind 2^31 bytes
    K2 = 65664
    w2 = torch.zeros(E, 33024, K2, dtype=torch.uint8, device="cuda")
    w2[1, -256:, :128] = w.view(torch.uint8).cuda()
    s2 = torch.ones(E, 258, K2 // 128, device="cuda")
    s2[1, -2:, 0] = ws.cuda()[:, 0]
    x2 = torch.zeros(300, K2, dtype=torch.uint8, device="cuda")
    x2[:, :128] = xd[:300]
    xs2 = torch.ones(K2 // 128, 300, device="cuda")
    xs2[0] = xsd[0, :300]
    y2 = torch.zeros(300, 33024, dtype=torch.bfloat16, device="cuda")
    call(kge, "kge_gemm_fp8_grouped", y2, x2, xs2, 300, w2, s2, torch.tensor([0, 150, 300], **I32), E, 300, 33024, K2, work, work.numel())
    held(y2[150:, -256:].cpu(), z[150:300], a[150:300], K2, fo.half_step(torch.bfloat16))
    assert (y2[:150] == 0).all() and (y2[150:, :-256] == 0).all()
    del w2
    # rows quantised from beyond 2^31 numbers
    K3, T3 = 131072, 16600
    big = torch.zeros(T3, K3, dtype=torch.bfloat16, device="cuda")
    big[-1] = torch.randn(K3, generator=g).to(torch.bfloat16)
    codes, scales = torch.zeros(T3, K3, dtype=torch.uint8, device="cuda"), torch.zeros(K3 // 128, T3, device="cuda")
    call(kge, "kge_fp8_quant", codes, scales, T3, big, K3, None, T3, K3)
    code, scale = fo.quantise(big[-1:].cpu(), 1)
    assert torch.equal(codes[-1].cpu().view(fo.E4M3).double(), code[0]) and torch.equal(scales[:, -1].cpu(), scale[0].float())
    assert not codes[:-1].any()


ALIGNED = [  # T, N, K: tiles of 256 columns, several a CTA; tiles of 128 cut along K over a cluster; pairs, whole and ragged; a column more, then seven
    (70, 19001, 144), (33, 19175, 144), (130, 30002, 144), (1, 4097, 2064), (64, 1001, 1040), (100, 3005, 1296), (9, 3, 528), (128, 6143, 528), (1030, 2049, 272), (2050, 1029, 400),
    (777, 4095, 144), (200, 1024, 400), (64, 2048, 528), (600, 4096, 144), (3, 40000, 144), (1, 4096, 2064)]


@pytest.mark.parametrize("T,N,K", ALIGNED)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_results_and_biases_at_any_address(kge, L, T, N, K, dtype):
    """y and the bias 0 to 7 elements behind a 16-byte boundary, rows of any alignment: sentinels around the result stay, and the bits do not depend on it."""
    dt, g = fo.DT[dtype], torch.Generator().manual_seed(T + N)
    x, xs, xn = quantised(g, T, K, 1)
    w, ws, wn = quantised(g, N, K, 128)
    b = torch.randn(N, generator=g).to(dt)
    xn, wn = xn.cuda(), wn.cuda()
    z, a = (xn @ wn.t()).cpu(), (xn.abs() @ wn.abs().t()).cpu()
    args = xs.t().contiguous().cuda(), T, w.cuda(), ws.cuda()
    xd, work = x.cuda(), workspace(L, T)
    for bias in (False, True):
        first = None
        for off in ((0, 1, 2, 7) if bias else (0, 1, 6)):
            room, broom = torch.full((T * N + 64,), 7.0, dtype=dt, device="cuda"), torch.full((N + 16,), math.nan, dtype=dt, device="cuda")
            broom[off:off + N] = b.cuda()
            call(kge, name("kge_gemm_fp8", dt), room[24 + off:], xd, *args, broom[off:] if bias else None, T, N, K, work, work.numel())
            y = room[24 + off:24 + off + T * N].view(T, N)
            assert (room[:24 + off] == 7).all() and (room[24 + off + T * N:] == 7).all()
            if first is None:
                first = y.clone()
                held(first.cpu(), z + b.double() if bias else z, a + b.double().abs() if bias else a, K, fo.half_step(dt))
            assert torch.equal(y, first), off


@pytest.mark.parametrize("sizes,N,K", [([5, 0, 1, 33], 137, 528), ([300, 2, 0, 33, 129], 515, 400), ([1] * 40, 4098, 144), ([60] * 20, 1283, 272), ([200, 31, 0, 257], 1001, 656),
                                       ([2, 1, 0, 3], 67, 2064)], ids=lambda v: str(v) if isinstance(v, int) else "x".join(map(str, v))[:24])
@pytest.mark.parametrize("off", [0, 1, 6])
def test_groups_with_rows_of_any_alignment(kge, L, sizes, N, K, off):
    g, E, T = torch.Generator().manual_seed(N), len(sizes), sum(sizes)
    x, xs, xn = quantised(g, T, K, 1)
    w, ws, wn = quantised(g, E * 128 * -(-N // 128), K, 128)
    w, wn = (v.unflatten(0, (E, -1))[:, :N].contiguous() for v in (w, wn))
    offsets = np.concatenate([[0], np.cumsum(sizes)])
    room = torch.full(((T + 9) * N + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
    work = workspace(L, T + 9)
    xd, xsd = torch.zeros(T + 9, K, dtype=torch.uint8, device="cuda"), torch.zeros(xs.shape[1], T + 9, device="cuda")
    xd[:T], xsd[:, :T] = x.cuda().view(torch.uint8), xs.t().cuda()
    call(kge, "kge_gemm_fp8_grouped", room[32 + off:], xd, xsd, T + 9, w.cuda(), ws.cuda(), torch.tensor(offsets, **I32), E, T + 9, N, K, work, work.numel())
    y = room[32 + off:32 + off + T * N].view(T, N).cpu()
    assert (room[:32 + off] == 7).all() and (room[32 + off + T * N:] == 7).all() and (work[:1024] == 0).all()
    for e in range(E):
        r = slice(offsets[e], offsets[e + 1])
        if sizes[e]:
            held(y[r], xn[r] @ wn[e].t(), xn[r].abs() @ wn[e].abs().t(), K, fo.half_step(torch.bfloat16))


@pytest.mark.parametrize("T,f,K", [(97, 128, 272), (128, 1024, 1040), (97, 896, 2064), (370, 640, 2064), (1112, 128, 1040), (65, 256, 1424), (100, 2304, 528), (120, 2944, 400)])
def test_gated_tiles_whose_sums_take_the_place_of_their_stages(kge, L, T, f, K):
    """More than 96 rows in tiles cut along K over 2 to 8 CTAs (and one of fewer): twice over, and after itself, with the same bits."""
    g = torch.Generator().manual_seed(T + f)
    x, xs, xn = quantised(g, T, K, 1)
    w, ws, wn = quantised(g, 2 * f, K, 128)
    work = workspace(L, T)
    args = x.cuda(), xs.t().contiguous().cuda(), T, w.cuda(), ws.cuda(), T, f, K, work, work.numel()
    out = [(torch.full((T + 1, f), 0x55, dtype=torch.uint8, device="cuda"), torch.full((f // 128, T), 9.0, device="cuda")) for _ in range(5)]
    for codes, scales in out:
        call(kge, "kge_gemm_fp8_silu_gate", codes, scales, T, *args)
    torch.cuda.synchronize()
    xn, wn = xn.cuda(), wn.cuda()
    codes, scales = out[0]
    held_gated(codes[:T].cpu().view(fo.E4M3), scales.cpu().t(), (xn @ wn.t()).cpu(), (xn.abs() @ wn.abs().t()).cpu(), K)
    for c, s in out:
        assert (c[T] == 0x55).all() and torch.equal(c, codes) and torch.equal(s, scales)


@pytest.mark.parametrize("dtype,T,K", [("bf16", 2400, 2080), ("fp16", 9500, 672), ("bf16", 4800, 1024), ("fp16", 1400, 3616), ("bf16", 9473, 544), ("bf16", 700, 7168)])
@pytest.mark.parametrize("form", ["plain", "strided", "gathered"])
def test_many_rows_bit_for_bit(kge, L, dtype, T, K, form):
    test_rows_are_quantised_bit_for_bit(kge, L, dtype, T, K, form)


@pytest.mark.parametrize("T,K", [(5, 4096), (2400, 2080), (9500, 672)])
def test_codes_at_any_16_bytes(kge, L, T, K):
    x = rows_of(torch.Generator().manual_seed(T), T, K, torch.bfloat16).cuda()
    out = []
    for off in (0, 16, 48):
        room, scales = torch.full((T * K + 96,), 0x55, dtype=torch.uint8, device="cuda"), torch.zeros(-(-K // 128), T, device="cuda")
        call(kge, "kge_fp8_quant", room[off:], scales, T, x, K, None, T, K)
        out.append((room[off:off + T * K].clone(), scales))
        assert (room[:off] == 0x55).all() and (room[off + T * K:] == 0x55).all()
    assert all(torch.equal(c, out[0][0]) and torch.equal(s, out[0][1]) for c, s in out)


@pytest.mark.parametrize("dtype,E,N,K", [("bf16", 7, 700, 2320), ("fp16", 40, 130, 1296), ("bf16", 1, 3000, 2064), ("fp16", 300, 65, 48), ("bf16", 2, 10100, 528)])
def test_weights_of_many_steps_bit_for_bit(kge, L, dtype, E, N, K):
    test_weights_are_quantised_bit_for_bit(kge, L, dtype, E, N, K)


@pytest.mark.parametrize("sizes,N,K", [([1], 64, 4240), ([5, 0, 1, 0, 0, 40], 136, 5136), ([33, 70], 520, 8208), ([0, 128, 3], 384, 4112), ([97, 0, 2, 31], 640, 4224), ([7] * 12, 256, 4608)],
                         ids=lambda v: str(v) if isinstance(v, int) else "x".join(map(str, v)))
@pytest.mark.parametrize("form", ["bf16", "fp16", "gated"])
@pytest.mark.parametrize("first,behind", [(0, 0), (3, 9)])
def test_groups_cut_along_k(kge, L, sizes, N, K, form, first, behind):
    test_grouped(kge, L, sizes, N, K, form, first, behind)
