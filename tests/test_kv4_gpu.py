"""The 4-bit key-value cache on the GPU: rows written and read back bit for bit, attention against 64 bits, tables of a step, and all of
them together as a serving loop uses them.

Tolerances.  u is half a step of the 16-bit type relative to the value, eps / 2 (bf16 2^-8, fp16 2^-11).
  Codes n - 8 are exact in the products, and so is q (but for what lies 2^-24 below its largest number in single-token requests).  Weights p s
  are rounded once, to float16 (2^-11) in single-token requests and at most to the 16-bit type (u) in prompts; what they are multiplied with is
  |n - 8| <= 8, so that costs 8 max s of it at most.  The result is rounded once, u |out|.  Scores and sums are in fp32: their errors stay below
  2^-13 of the weights here.
  (Prompts round them to float16 too, which is less than u 8 max s; test_kv4_rows_gpu.py holds both to the roundings alone.)
  In the 2-norm the roundings are independent, each of at most u / sqrt(3) in the mean square: result and weights together sqrt(2 / 3) u =
  0.82 u where s (n - 8) is as large as the values (their ends lie about zero), held to 1.2 (u + 2^-11).
"""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import kv4_oracle as ko

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


def randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g) * std


def cos_sin(hd, n, dt, theta=10000.0):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * theta ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)[None]
    return torch.cat([ang.cos(), ang.sin()], -1).to(dt)


def turned(x, cs):
    """[T, heads, hd] 16-bit rows turned in fp32 and rounded once."""
    c, s = cs.float()[:, None].chunk(2, -1)
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)


# ------------------------------------------------------------------------------------------------------- rows of the cache

WRITES = [  # dtype, hd, H, KV, block, T
    ("bf16", 128, 4, 2, 16, 1), ("bf16", 128, 32, 8, 64, 7), ("fp16", 128, 5, 1, 32, 33), ("bf16", 64, 3, 3, 16, 50), ("fp16", 64, 7, 1, 128, 19),
    ("fp16", 64, 1, 1, 16, 2), ("bf16", 64, 32, 8, 16, 21), ("bf16", 128, 1, 1, 256, 40), ("fp16", 128, 8, 8, 64, 100),
    ("fp16", 64, 4, 1, 16, 4), ("bf16", 64, 8, 1, 32, 129), ("fp16", 128, 4, 2, 16, 131), ("bf16", 128, 6, 1, 64, 2)]


@pytest.mark.parametrize("dtype,hd,H,KV,bs,T", WRITES)
@pytest.mark.parametrize("rotate", [True, False])
def test_rows_are_written_bit_for_bit(kge, L, dtype, hd, H, KV, bs, T, rotate):
    dt, g = ko.DT[dtype], torch.Generator().manual_seed(T * 7 + hd)
    x = randn(g, T, H + 2 * KV, hd).to(dt)
    cs = cos_sin(hd, 300, dt)
    pos = torch.randint(0, 300, (T,), generator=g)
    blocks = T // bs + 3
    slots = (torch.randperm(blocks * bs, generator=g)[:T]).long()
    slots[max(1, T // 2)::5] = -1                                           # rows for no cache
    want = ko.Cache(blocks, KV, hd, bs, dt, fill=0xA5)              # what is not written stays
    y = torch.cat([turned(x[:, :H + KV], cs[pos]), x[:, H + KV:]], 1) if rotate else x
    want.put(y[:, H:H + KV], y[:, H + KV:], slots.tolist())
    qkv, cache = x.reshape(T, -1).cuda(), torch.full(want.data.shape, 0xA5, dtype=torch.uint8, device="cuda")
    assert cache.numel() == L.kge_kv4_cache_bytes(blocks, KV, hd, bs)
    width = H * hd + 24
    q = torch.full((T, width), 7.0, dtype=dt, device="cuda")
    call(kge, name("kge_rope_kv4write", dt), q, width, cache, qkv, cs.cuda() if rotate else None, pos.int().cuda(), slots.cuda(), T, H, KV, hd, bs)
    torch.cuda.synchronize()
    assert torch.equal(q[:, :H * hd].cpu().view(torch.int16), y[:, :H].reshape(T, -1).view(torch.int16))
    assert (q[:, H * hd:] == 7).all() and torch.equal(qkv.cpu(), x.reshape(T, -1))
    assert torch.equal(cache.cpu(), torch.from_numpy(want.data))
    # q in place of the packed buffer gives the same, and leaves its keys and values alone
    cache.fill_(0xA5)
    call(kge, name("kge_rope_kv4write", dt), qkv, qkv.shape[1], cache, qkv, cs.cuda() if rotate else None, pos.int().cuda(), slots.cuda(), T, H, KV, hd, bs)
    torch.cuda.synchronize()
    assert torch.equal(cache.cpu(), torch.from_numpy(want.data))
    assert torch.equal(qkv.cpu(), torch.cat([y[:, :H], x[:, H:]], 1).reshape(T, -1))
    # and back: low + scale code, rounded once
    k, v = (torch.full((T, KV, hd), 9.0, dtype=dt, device="cuda") for _ in range(2))
    call(kge, name("kge_kv4_read", dt), k, v, cache, slots.cuda(), T, KV, hd, bs)
    torch.cuda.synchronize()
    there = slots >= 0
    for h in range(KV):
        for got, ref, src in zip((k, v), want.get(slots[there].tolist(), h), (y[:, H + h], y[:, H + KV + h])):
            assert torch.equal(got[there.cuda(), h].cpu(), ref.float().to(dt))
            step = (src.float().amax(1) - src.float().amin(1))[there, None] / 15 * (1 + 2 * ko.half_step(dt))
            assert (ref - src[there].double()).abs().le(step / 2 + 1e-30).all()
    assert (k[~there.cuda()] == 0).all() and (v[~there.cuda()] == 0).all()


SPECIAL = {
    "zeros": lambda x, big: x * 0, "constant": lambda x, big: x * 0 + 3.25, "negative zero": lambda x, big: x * 0 - 0.0, "one nan": lambda x, big: _set(x, math.nan),
    "inf": lambda x, big: _set(x, math.inf), "minus inf": lambda x, big: _set(x, -math.inf), "largest": lambda x, big: _set(x * 0, big),
    "both ends": lambda x, big: _set(_set(x * 0, big), -big, 3), "tiny": lambda x, big: x * 1e-7, "denormal": lambda x, big: x * 0 + (torch.arange(x.shape[-1]) % 3) * 6e-8,
    "offset": lambda x, big: x * 0.01 + 100, "one large": lambda x, big: _set(x, 300.0)}


def _set(x, v, at=11):
    x = x.clone()
    x[..., at] = v
    return x


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", sorted(SPECIAL))
def test_rows_of_special_numbers(kge, L, dtype, hd, kind):
    """Infinities, NaN, no range, and a range of the whole type: a finite row reads back within half its scale and finite, others as NaN."""
    dt = ko.DT[dtype]
    g = torch.Generator().manual_seed(3)
    x = randn(g, 5, 3, hd).to(dt)
    x[2, 1] = SPECIAL[kind](x[2, 1].float(), torch.finfo(dt).max).to(dt)
    x[3, 2] = SPECIAL[kind](x[3, 2].float(), torch.finfo(dt).max).to(dt)
    slots = torch.tensor([3, 0, 9, 20, 14])
    want = ko.Cache(2, 1, hd, 16, dt)
    want.put(x[:, 1:2], x[:, 2:], slots.tolist())
    cache, q = torch.zeros(want.data.shape, dtype=torch.uint8, device="cuda"), torch.zeros(5, hd, dtype=dt, device="cuda")
    call(kge, name("kge_rope_kv4write", dt), q, hd, cache, x.reshape(5, -1).cuda(), None, None, slots.cuda(), 5, 1, 1, hd, 16)
    k, v = (torch.zeros(5, 1, hd, dtype=dt, device="cuda") for _ in range(2))
    call(kge, name("kge_kv4_read", dt), k, v, cache, slots.cuda(), 5, 1, hd, 16)
    torch.cuda.synchronize()
    assert torch.equal(cache.cpu(), torch.from_numpy(want.data))
    for got, src in ((k[:, 0].cpu(), x[:, 1]), (v[:, 0].cpu(), x[:, 2])):
        span = src.double().amax(1, keepdim=True) - src.double().amin(1, keepdim=True)
        fine = torch.isfinite(span.float())[:, 0]
        assert torch.isnan(got[~fine]).all() and torch.isfinite(got[fine]).all()
        # half a scale (rounded up to the type: 1 + 2 u, or a least step of its denormals more), and the 16-bit result's own rounding
        least = 2.0 ** -24 if dt == torch.float16 else 2.0 ** -133
        slack = (span / 15 * (1 + 2 * ko.half_step(dt)) + least) / 2 + ko.half_step(dt) * src.double().abs().amax(1, keepdim=True) * 1.1 + least
        assert ((got.double() - src.double()).abs() <= slack)[fine].all()


# ------------------------------------------------------------------------------------------------------------- attention

def setup(dtype, hd, H, KV, bs, lens, news, seed=0, std=1.0, extra_rows=0, stride_pad=0, spare=2):
    """A batch over a filled cache; every page's unused rows and the blocks of no request hold NaN rows."""
    dt, g = ko.DT[dtype], torch.Generator().manual_seed(1000 + seed)
    per = [-(-n // bs) for n in lens]
    blocks = sum(per) + spare
    order = (torch.randperm(blocks - 1, generator=g) + 1).tolist()
    table = np.zeros((len(lens), max(max(per), 1) + 1), dtype=np.int32)
    cache = ko.Cache(blocks, KV, hd, bs, dt, fill=0xFF)             # 0xffff is NaN in both types
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    for b, n in enumerate(lens):
        if n:
            slots = [int(table[b, j // bs]) * bs + j % bs for j in range(n)]
            cache.put(randn(g, n, KV, hd, std=std).to(dt), randn(g, n, KV, hd, std=std).to(dt), slots)
    T = sum(news)
    q = randn(g, T + extra_rows, H * hd + stride_pad, std=std).to(dt)
    qsl = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    return dict(dt=dt, cache=cache, table=table, q=q, qsl=qsl, lens=list(lens), H=H, KV=KV, hd=hd, bs=bs, T=T)


def attend(kge, s, window=0, first=0, scale=None, maxq=None, maxc=None, out=None, data=None, stream=None, ws=None):
    H, KV, hd = s["H"], s["KV"], s["hd"]
    news = np.diff(s["qsl"])
    q = s["q"].cuda()
    out = torch.full((q.shape[0], H * hd), 5.0, dtype=s["dt"], device="cuda") if out is None else out
    n = kge.lib().kge_attn_kv4_workspace_bytes(H, KV, hd)
    ws = torch.full((max(n, 16),), 0xFF, dtype=torch.uint8, device="cuda") if ws is None else ws
    data = s["cache"].tensor() if data is None else data
    call(kge, name("kge_paged_attn_kv4", s["dt"]), out, q, q.shape[1], data, torch.from_numpy(s["table"]).cuda(), s["table"].shape[1],
         torch.tensor(s["lens"], **I32), torch.from_numpy(s["qsl"]).cuda(), len(s["lens"]), q.shape[0], maxq or max(1, int(news.max())), maxc or max(1, max(s["lens"])), H, KV, hd,
         s["bs"], scale or hd ** -0.5, window, first, ws, ws.numel(), stream=stream)
    torch.cuda.synchronize()
    return out


def check(s, out, window=0, first=0, scale=None, norm=True):
    H, hd, T, u = s["H"], s["hd"], s["T"], ko.half_step(s["dt"])
    ref, size, reach = ko.attention(s["cache"], s["q"][:T, :H * hd].reshape(T, H, hd), s["table"], s["lens"], s["qsl"], H, scale or hd ** -0.5, window, first)
    got = out[:T].cpu().double().reshape(T, H, hd)
    assert (out[T:] == 5).all()                                     # rows behind the last request
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    fine = ~torch.isnan(ref)
    news = np.diff(s["qsl"])
    single = torch.from_numpy(np.repeat(news == 1, news)) & (H // s["KV"] <= 16)
    params = s["cache"].data[..., 16 * hd:].reshape(-1, 4)[:, :2].copy()
    scales = torch.from_numpy(params).view(s["dt"]).double()
    top = float(scales[torch.isfinite(scales)].max()) if torch.isfinite(scales).any() else 0.0
    weight = torch.where(single, 2.0 ** -11, u)[:, None, None]
    loose = (weight * 1.01 + 2 ** -13) * 8 * top + 2 ** -13 * size
    tol = u * ref.abs() * 1.01 + loose + 1e-12
    err = (got - ref).abs()
    assert (err <= tol)[fine].all(), (float((err / tol)[fine].max()), float(err[fine].max()))
    if norm and int(fine.sum()) >= 1000:
        ref, got = (torch.where(fine, x, 0.0) for x in (ref, got))
        assert (got - ref).norm() <= 1.2 * (u + 2 ** -11) * ref.norm(), float((got - ref).norm() / ref.norm() / u)


LENS = [1, 2, 3, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 100, 127, 129]
DECODE = [  # dtype, hd, H, KV, block, lengths
    ("bf16", 128, 8, 2, 16, LENS), ("fp16", 64, 8, 2, 16, LENS), ("bf16", 64, 3, 3, 32, LENS), ("fp16", 128, 6, 2, 64, LENS), ("bf16", 128, 8, 1, 128, LENS),
    ("bf16", 128, 9, 1, 16, [1, 40, 130]), ("fp16", 64, 16, 1, 32, [5, 77]), ("bf16", 64, 24, 2, 16, [333, 12]), ("fp16", 128, 32, 2, 64, [70, 200, 1]),
    # beyond the line for cut contexts
    ("bf16", 128, 4, 1, 64, [700, 1, 33, 512, 1500]), ("fp16", 64, 8, 4, 16, [900]), ("bf16", 64, 16, 1, 32, [2000, 600]), ("fp16", 128, 13, 1, 16, [1111, 40]),
    ("bf16", 128, 7, 7, 256, [555, 640, 3])]


@pytest.mark.parametrize("dtype,hd,H,KV,bs,lens", DECODE)
@pytest.mark.parametrize("window,first", [(0, 0), (1, 0), (7, 3), (40, 0), (64, 17), (100, 64), (3000, 5)])
def test_single_tokens(kge, L, dtype, hd, H, KV, bs, lens, window, first):
    s = setup(dtype, hd, H, KV, bs, lens, [1] * len(lens), seed=hd + H, extra_rows=2, stride_pad=8 * (H % 3))
    check(s, attend(kge, s, window, first), window, first)


PROMPTS = [  # dtype, hd, H, KV, block, lengths, rows
    ("bf16", 128, 4, 1, 16, [5, 64, 65, 130], [5, 64, 65, 130]), ("fp16", 64, 8, 2, 32, [2, 33, 128, 200], [2, 33, 100, 77]), ("bf16", 64, 3, 3, 64, [150, 300], [150, 129]),
    ("fp16", 128, 8, 1, 16, [90, 17], [90, 17]), ("bf16", 128, 5, 1, 128, [333, 40], [51, 40]), ("bf16", 64, 40, 2, 16, [70, 9, 33], [70, 1, 3]),
    ("fp16", 128, 32, 1, 64, [100, 200, 1], [1, 64, 1]), ("bf16", 128, 2, 2, 32, [700], [450]), ("fp16", 64, 6, 1, 16, [260, 262, 265], [260, 262, 265])]


@pytest.mark.parametrize("dtype,hd,H,KV,bs,lens,news", PROMPTS)
@pytest.mark.parametrize("window,first", [(0, 0), (1, 0), (7, 3), (64, 0), (65, 70), (100, 4), (1000, 5)])
def test_prompts(kge, L, dtype, hd, H, KV, bs, lens, news, window, first):
    s = setup(dtype, hd, H, KV, bs, lens, news, seed=hd + H + 1, extra_rows=3)
    check(s, attend(kge, s, window, first), window, first)


@pytest.mark.parametrize("dtype,hd,H,KV,bs,lens,news", [
    ("bf16", 64, 128, 1, 4096, [5000, 1, 70], [1, 1, 3]),                   # 128 heads on one, the largest blocks
    ("fp16", 128, 128, 128, 16, [37, 9], [1, 9]),                           # as many kv heads
    ("bf16", 128, 34, 2, 2048, [2049, 300], [2, 1]),                        # one head more than the single-token kernel takes
    ("fp16", 64, 16, 16, 4096, [4097], [1]), ("bf16", 128, 127, 127, 32, [33, 65], [1, 20])])
@pytest.mark.parametrize("window,first", [(2 ** 31 - 1, 2 ** 31 - 1), (33, 40)])
def test_the_largest_sizes(kge, L, dtype, hd, H, KV, bs, lens, news, window, first):
    """Heads, blocks, windows and bounds at the ends of their ranges, rows of q further apart than they are long."""
    s = setup(dtype, hd, H, KV, bs, lens, news, seed=31, extra_rows=2, stride_pad=40)
    check(s, attend(kge, s, window, first, maxq=70000, maxc=2 ** 31 - 1), window, first)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("window,first", [(0, 0), (50, 4)])
def test_mixed_batches(kge, L, dtype, window, first):
    """Decode rows, prompt chunks, requests without rows (with and without keys) and one without keys, in one call."""
    lens, news = [40, 0, 130, 33, 0, 300, 1, 20, 90], [1, 0, 100, 1, 1, 37, 1, 0, 2]
    s = setup(dtype, 128, 8, 2, 16, lens, news, seed=5, extra_rows=4)
    out = attend(kge, s, window, first, maxq=120, maxc=1000)
    check(s, out, window, first)
    assert (out[s["qsl"][4]] == 0).all()
    assert torch.equal(out, attend(kge, s, window, first, maxq=120, maxc=1000))          # the same bits again


def test_rows_before_the_first_key(kge, L):
    """A length below a request's rows: the first ones have no key, and are zeros."""
    for H in (4, 40):                                               # 40 heads: single tokens go with the prompts
        s = setup("bf16", 64, H, 1, 16, [3, 0, 80], [8, 1, 2], seed=8)
        out = attend(kge, s)
        check(s, out)
        assert (out[:5] == 0).all() and (out[8] == 0).all() and (out[5:8] != 0).any()


@pytest.mark.parametrize("H,KV,hd", [(8, 2, 128), (6, 6, 64), (40, 2, 64)])
@pytest.mark.parametrize("window,first", [(0, 0), (30, 2)])
def test_nan_rows_reach_those_who_see_them_only(kge, L, H, KV, hd, window, first):
    lens, news = [100, 70, 200, 64], [40, 1, 90, 64]
    s = setup("bf16", hd, H, KV, 16, lens, news, seed=9)
    g = torch.Generator().manual_seed(1)
    for b, j in ((0, 80), (0, 97), (1, 1), (1, 30), (2, 150), (3, 0), (3, 63)):       # keys and values with a NaN or an infinity
        slot = int(s["table"][b, j // 16]) * 16 + j % 16
        k, v = randn(g, 1, KV, hd).bfloat16(), randn(g, 1, KV, hd).bfloat16()
        (k if j % 2 else v)[0, KV - 1, j % hd] = math.nan if j % 4 else math.inf
        s["cache"].put(k, v, [slot])
    out = attend(kge, s, window, first)
    check(s, out, window, first)
    assert torch.isnan(out).any() and not torch.isnan(out).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_large_and_small_numbers(kge, L, dtype):
    """Scales far apart within one context, steep scores, constant values: the weights' reference has to follow both."""
    dt = ko.DT[dtype]
    s = setup(dtype, 128, 4, 1, 16, [300, 700, 90], [1, 1, 1], seed=11)
    g = torch.Generator().manual_seed(2)
    big = 1e4 if dt == torch.float16 else 1e20
    for b, n in enumerate(s["lens"]):
        slots = [int(s["table"][b, j // 16]) * 16 + j % 16 for j in range(n)]
        size = torch.exp(torch.empty(n, 1, 1).uniform_(math.log(1e-4), math.log(big), generator=g))
        size[::7] = 0
        s["cache"].put((randn(g, n, 1, 128) * (3 if b else 30)).to(dt), (randn(g, n, 1, 128) * size + (5.0 if b == 2 else 0.0)).clamp(-6e4 if dt == torch.float16 else -1e30, 6e4 if dt == torch.float16 else 1e30).to(dt), slots)
    out = attend(kge, s)
    ref, size, reach = ko.attention(s["cache"], s["q"].reshape(3, 4, 128), s["table"], s["lens"], s["qsl"], 4, 128 ** -0.5)
    got, u = out.cpu().double().reshape(3, 4, 128), ko.half_step(dt)
    # weights round by 2^-11 of p s |c'|, and p s |c'| <= 8 p s <= 2 (p |v| at the row's ends): of the sum of the rows' largest |p v|
    most = size.amax(-1, keepdim=True)
    # fp32 scores of up to `reach`: 130 roundings of 2^-24 of it at most
    assert ((got - ref).abs() <= u * ref.abs() + (2 ** -10 + 2 * 130 * 2.0 ** -24 * reach) * 8 * most).all()
    assert torch.isfinite(got).all()


def test_q_beyond_float16(kge, L):
    """bf16 queries whose numbers no float16 holds, heads of one group far apart, a head of zeros, and one with an infinity beside it."""
    s = setup("bf16", 128, 4, 1, 16, [50, 600], [1, 1], seed=12)
    scale = 1e-9
    q = s["q"].reshape(2, 4, 128)
    q[:, 0] *= 3e9
    q[:, 1] *= 1e7
    q[:, 2] = 0
    out = attend(kge, s, scale=scale)
    check(s, out, scale=scale, norm=False)
    q[1, 3, 5] = math.inf
    again = attend(kge, s, scale=scale).reshape(2, 4, 128)
    assert torch.equal(again[0], out.reshape(2, 4, 128)[0]) and torch.equal(again[1, :3], out.reshape(2, 4, 128)[1, :3])
    assert torch.isnan(again[1, 3]).any()


@pytest.mark.parametrize("hd,H,KV", [(128, 4, 1), (64, 6, 2)])
@pytest.mark.parametrize("window,first", [(0, 0), (90, 3)])
def test_prompts_of_numbers_far_apart(kge, L, hd, H, KV, window, first):
    """bf16 prompts whose queries, keys and values no float16 holds: 64-key tiles 10^24 apart (within one, 100), rows of q 10^9 apart, rows of
    zeros, and pages that hold the largest numbers behind the last key and in front of the window."""
    lens, news = [400, 150, 70], [90, 150, 3]
    s = setup("bf16", hd, H, KV, 16, lens, news, seed=21)
    g = torch.Generator().manual_seed(22)
    for b, n in enumerate(lens):
        end = -(-n // 16) * 16
        slots = [int(s["table"][b, j // 16]) * 16 + j % 16 for j in range(end)]
        within = 10 ** torch.empty(end, 1, 1).uniform_(-1, 1, generator=g)
        tiles = (10 ** torch.empty(2, end // 64 + 1).uniform_(-12, 12, generator=g)).repeat_interleave(64, 1)[:, :end, None, None]
        k, v = randn(g, end, KV, hd) * within, randn(g, end, KV, hd) * within * tiles[1]
        k[torch.arange(end) // 64 % 3 == 0] *= 1e-10
        k[n:], v[n:] = randn(g, end - n, KV, hd) * 1e37, randn(g, end - n, KV, hd) * 1e37
        v[5:5 + 64] *= 0 if b == 1 else 1
        if window and b == 0:
            k[first:n - news[b] - window + 1], v[first:n - news[b] - window + 1] = 1e37, -1e37
        s["cache"].put(k.bfloat16(), v.bfloat16(), slots)
    q = s["q"][:, :H * hd].reshape(-1, H, hd)
    q *= 10 ** torch.empty(q.shape[0], H, 1).uniform_(-9, 0, generator=g) * 1e12
    q[3] = 0
    scale = hd ** -0.5 * 1e-13
    out = attend(kge, s, window, first, scale=scale)
    T = s["T"]
    ref, size, reach = ko.attention(s["cache"], s["q"][:T, :H * hd].reshape(T, H, hd), s["table"], s["lens"], s["qsl"], H, scale, window, first)
    got, u = out[:T].cpu().double().reshape(T, H, hd), ko.half_step(torch.bfloat16)
    # 2^-11 each for weights and values, and twice that of the scores' sum |q k| scale for the keys.  Besides, a tile's numbers end at 2^-16 of its
    # largest scale, here 150 times a row's own at most, which is max |v| / 7.5 at most: 2^-11.6 max |v|, and sum p max |v| < 3 max sum p |v|, so
    # 2^-10 of that; of a score 2^-16 150 / 7.5 max |k| sum |q| scale, with max |k| < 4 of the mean |k|: 2^-9.6 of its sum, twice that for the weights
    assert ((got - ref).abs() <= u * ref.abs() * 1.01 + 2 ** -11 * (2 + 8 * reach) * size + 2 ** -10 * size.amax(-1, keepdim=True)).all()
    q[7, 1, 3] = math.inf                                              # a row that cannot be multiplied, beside others
    again = attend(kge, s, window, first, scale=scale)[:T].cpu().reshape(T, H, hd)
    rest = torch.ones(T, H, dtype=torch.bool)
    rest[7, 1] = False
    assert torch.equal(again[rest], out[:T].cpu().reshape(T, H, hd)[rest]) and torch.isnan(again[7, 1]).any()


def test_offsets_beyond_32_bits(kge, L):
    """Blocks whose bytes lie past 2^31 and 2^32 of the cache."""
    KV, hd, bs = 8, 128, 64
    per = KV * bs * (hd + 8)
    blocks = (1 << 32) // per + 40
    s = setup("bf16", hd, 8, KV, bs, [200, 70], [1, 70], seed=13)
    data = torch.zeros(blocks * per, dtype=torch.uint8, device="cuda")
    small, far = s["cache"].tensor().reshape(-1, per), {}
    for b in range(2):
        for i in range(s["table"].shape[1]):
            if s["table"][b, i]:
                far[int(s["table"][b, i])] = ((1 << 31) if b else (1 << 32)) // per + 1 + 3 * i
    for old, new in far.items():
        data.view(-1, per)[new] = small[old]
    want = attend(kge, s)
    s2 = dict(s, table=np.array([[far.get(int(x), 0) for x in row] for row in s["table"]], dtype=np.int32))
    assert torch.equal(attend(kge, s2, data=data), want)
    # rows there are written and read as well
    g = torch.Generator().manual_seed(4)
    x = randn(g, 2, 8 + 16, hd).bfloat16().cuda()
    slots = torch.tensor([(blocks - 1) * bs + 63, ((1 << 31) // per + 2) * bs + 5], device="cuda")
    q, k, v = torch.empty(2, 8 * hd, dtype=torch.bfloat16, device="cuda"), *(torch.empty(2, KV, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    call(kge, "kge_rope_kv4write", q, 8 * hd, data, x, None, None, slots, 2, 8, KV, hd, bs)
    call(kge, "kge_kv4_read", k, v, data, slots, 2, KV, hd, bs)
    small = torch.zeros(2 * per, dtype=torch.uint8, device="cuda")
    k2, v2 = torch.empty_like(k), torch.empty_like(v)
    call(kge, "kge_rope_kv4write", q, 8 * hd, small, x, None, None, slots % bs, 2, 8, KV, hd, bs)
    call(kge, "kge_kv4_read", k2, v2, small, slots % bs, 2, KV, hd, bs)
    torch.cuda.synchronize()
    assert torch.equal(k, k2) and torch.equal(v, v2) and (k != 0).any()


def test_many_requests(kge, L):
    """More requests than one launch takes, some without rows."""
    r = np.random.default_rng(3)
    lens = r.integers(1, 40, 1500).tolist()
    news = (r.random(1500) < 0.9).astype(int).tolist()
    s = setup("bf16", 64, 2, 1, 16, lens, news, seed=14, extra_rows=1)
    check(s, attend(kge, s))
    check(s, attend(kge, s, 9, 2, maxc=100000), 9, 2)               # (through the cut contexts)


# ------------------------------------------------------------------------------------------------------- tables of a step

def run_maps(kge, table, cached, new, free, first, T, bs, in_place=False):
    t = torch.from_numpy(table.copy()).cuda()
    c, n, f = (torch.tensor(x, **I32) for x in (cached, new, free if len(free) else [0]))
    B = len(cached)
    lens, qsl, pos = c if in_place else torch.full((B,), -7, **I32), torch.full((B + 1,), -7, **I32), torch.full((T + 3,), -7, **I32)
    slots, counts = torch.full((T + 3,), -7, dtype=torch.int64, device="cuda"), torch.full((4,), -7, **I32)
    if in_place:
        counts[2] = first
    at = counts[2:3] if in_place else torch.tensor([first], **I32)
    call(kge, "kge_step_maps", t, table.shape[1], lens, qsl, pos, slots, counts, c, n, f, len(free), at, B, T, bs)
    torch.cuda.synchronize()
    assert (pos[T:] == -7).all() and (slots[T:] == -7).all()
    return t.cpu().numpy(), lens.tolist(), qsl.tolist(), pos[:T].tolist(), slots[:T].tolist(), counts.tolist()


def random_maps(seed):
    r = np.random.default_rng(seed)
    bs = int(r.choice([1, 16, 32, 64, 256]))
    B = int(r.choice([1, 2, 31, 33, 200, 513, 1000, 8192] if seed % 5 == 0 else [1, 5, 40, 100, 515]))
    M = int(r.integers(1, 12))
    cached = np.where(r.random(B) < 0.2, 0, r.integers(0, M * bs + 1, B)).tolist()
    new = np.where(r.random(B) < 0.6, 1, r.integers(0, 3 * bs + 2, B)).tolist()
    table = r.integers(1, 1 << 20, (B, M)).astype(np.int32)
    need = sum(new) // bs + B
    free = r.permutation(int(need * r.choice([0.3, 1.5])) + 2)[: int(need * r.choice([0.3, 1.5])) + 2].astype(np.int32).tolist()
    T = max(1, int(sum(new) * r.choice([0.5, 1.0, 1.1])) + int(r.integers(0, 4)))
    return table, cached, new, free, int(r.integers(0, 3)), T, bs


@pytest.mark.parametrize("seed", range(30))
@pytest.mark.parametrize("in_place", [False, True])
def test_maps_of_random_steps(kge, L, seed, in_place):
    a = random_maps(seed)
    got, want = run_maps(kge, *a, in_place=in_place), ko.maps(*a)
    assert (got[0] == want[0]).all()
    for g, w in zip(got[1:], want[1:]):
        assert g == w


@pytest.mark.parametrize("case", [
    ([[5, 6]], [0], [0], [], 0, 4, 16), ([[5, 6]], [16], [5], [9], 0, 5, 16), ([[5, 6]], [30], [50], [9], 0, 100, 16), ([[5, 6]], [-3], [-1], [9], -2, 2, 16),
    ([[5, 6], [7, 8]], [16, 3], [1, 1], [], 0, 2, 16), ([[5, 6], [7, 8]], [10, 20], [2 ** 31 - 1, 2 ** 31 - 1], [1, 2, 3], 1, 9, 16), ([[5, 6]], [99], [4], [1], 5, 3, 16),
    ([[5, 0, 0]], [16], [40], [3], 0, 64, 16), ([[5, 0], [6, 0], [7, 0]], [16, 16, 16], [1, 0, 1], [4], 0, 3, 16), ([[1]], [0], [1], [7], 0, 0, 1)])
def test_maps_at_their_limits(kge, L, case):
    table, *rest = case
    a = (np.array(table, dtype=np.int32), *rest)
    got, want = run_maps(kge, *a), ko.maps(*a)
    assert (got[0] == want[0]).all()
    assert got[1:] == tuple(want[1:])


# ---------------------------------------------------------------------------------------------------------- all together

class Loop:
    """What a serving loop keeps on the GPU: pool, tables, free list; a step is maps, write and attention of one layer."""

    def __init__(self, kge, dt, H, KV, hd, bs, B, T, max_blocks, blocks):
        self.kge, self.dt, self.H, self.KV, self.hd, self.bs, self.B, self.T, self.max_blocks = kge, dt, H, KV, hd, bs, B, T, max_blocks
        g = torch.Generator().manual_seed(6)
        self.free = (torch.randperm(blocks - 1, generator=g) + 1).to(**I32)
        self.table = torch.zeros(B, max_blocks, **I32)
        self.lens, self.qsl, self.pos, self.counts = torch.zeros(B, **I32), torch.zeros(B + 1, **I32), torch.zeros(T, **I32), torch.zeros(4, **I32)
        self.slots, self.new = torch.zeros(T, dtype=torch.int64, device="cuda"), torch.zeros(B, **I32)
        self.cache = torch.full((kge.lib().kge_kv4_cache_bytes(blocks, KV, hd, bs),), 0xFF, dtype=torch.uint8, device="cuda")
        self.cs = cos_sin(hd, max_blocks * bs, dt).cuda()
        self.qkv = torch.zeros(T, (H + 2 * KV) * hd, dtype=dt, device="cuda")
        self.q, self.out = (torch.zeros(T, H * hd, dtype=dt, device="cuda") for _ in range(2))
        self.ws = torch.empty(kge.lib().kge_attn_kv4_workspace_bytes(H, KV, hd), dtype=torch.uint8, device="cuda")

    def step(self, window=0, first=0, maxq=None, stream=None):
        k, H, KV, hd, bs = self.kge, self.H, self.KV, self.hd, self.bs
        call(k, "kge_step_maps", self.table, self.max_blocks, self.lens, self.qsl, self.pos, self.slots, self.counts, self.lens, self.new, self.free, self.free.numel(),
             self.counts[2:3], self.B, self.T, bs, stream=stream)
        call(k, name("kge_rope_kv4write", self.dt), self.q, H * hd, self.cache, self.qkv, self.cs, self.pos, self.slots, self.T, H, KV, hd, bs, stream=stream)
        call(k, name("kge_paged_attn_kv4", self.dt), self.out, self.q, H * hd, self.cache, self.table, self.max_blocks, self.lens, self.qsl, self.B, self.T, maxq or self.T,
             self.max_blocks * bs, H, KV, hd, bs, hd ** -0.5, window, first, self.ws, self.ws.numel(), stream=stream)


class Mirror:
    """The same loop on the CPU, from the definitions."""

    def __init__(self, loop):
        self.l = loop
        self.cache = ko.Cache(loop.cache.numel() // (loop.KV * loop.bs * (loop.hd + 8)), loop.KV, loop.hd, loop.bs, loop.dt, fill=0xFF)
        self.table, self.lens, self.first = np.zeros((loop.B, loop.max_blocks), dtype=np.int32), [0] * loop.B, 0

    def step(self, new, qkv, window, first):
        l = self.l
        H, KV, hd = l.H, l.KV, l.hd
        self.table, self.lens, qsl, pos, slots, counts = ko.maps(self.table, self.lens, new, l.free.cpu().numpy(), self.first, l.T, l.bs)
        self.first = counts[2]
        x = qkv.reshape(l.T, H + 2 * KV, hd)
        y = turned(x[:, :H + KV], l.cs.cpu()[torch.tensor(pos)])
        self.cache.put(y[:, H:], x[:, H + KV:], slots)
        return dict(cache=self.cache, table=self.table, lens=self.lens, qsl=np.array(qsl), q=y[:, :H].reshape(l.T, -1), H=H, KV=KV, hd=hd, bs=l.bs, T=qsl[-1], dt=l.dt)


STEPS = [[5, 40, 0, 17], [1, 1, 30, 1], [1, 1, 1, 1], [1, 1, 1, 1], [1, 0, 20, 1], [1, 1, 1, 1]]


@pytest.mark.parametrize("dtype,H,KV,hd,bs", [("bf16", 8, 2, 128, 16), ("fp16", 6, 2, 64, 32)])
@pytest.mark.parametrize("window,first", [(0, 0), (24, 3)])
def test_a_run_of_steps(kge, L, dtype, H, KV, hd, bs, window, first):
    """Prompts, mixed and decode steps over a growing cache; lengths and tables never leave the GPU."""
    loop = Loop(kge, ko.DT[dtype], H, KV, hd, bs, 4, 64, 8, 30)
    mirror, g = Mirror(loop), torch.Generator().manual_seed(7)
    for new in STEPS:
        qkv = randn(g, 64, (H + 2 * KV) * hd).to(loop.dt)
        loop.qkv.copy_(qkv)
        loop.new.copy_(torch.tensor(new))
        loop.out.fill_(5)
        loop.step(window, first)
        torch.cuda.synchronize()
        s = mirror.step(new, qkv, window, first)
        assert loop.lens.tolist() == s["lens"] and loop.qsl.tolist() == s["qsl"].tolist()
        assert torch.equal(loop.q[:s["T"]].cpu(), s["q"][:s["T"]])
        check(s, loop.out, window, first)
    assert torch.equal(loop.cache.cpu().view(-1), torch.from_numpy(mirror.cache.data).view(-1))


def test_a_captured_step_is_replayed_with_other_lengths(kge, L):
    """One graph of maps, write and attention on a stream of its own serves prompts and decode steps alike."""
    H, KV, hd, bs = 8, 2, 128, 16
    side = torch.cuda.Stream()
    loop = Loop(kge, torch.bfloat16, H, KV, hd, bs, 4, 64, 8, 30)
    with torch.cuda.stream(side):
        loop.step(24, 3, stream=side)                               # (nothing new: no rows)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            loop.step(24, 3, stream=torch.cuda.current_stream())
    mirror, g = Mirror(loop), torch.Generator().manual_seed(7)
    for new in STEPS:
        qkv = randn(g, 64, (H + 2 * KV) * hd).to(loop.dt)
        loop.qkv.copy_(qkv)
        loop.new.copy_(torch.tensor(new))
        loop.out.fill_(5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        s = mirror.step(new, qkv, 24, 3)
        assert loop.lens.tolist() == s["lens"]
        check(s, loop.out, 24, 3)


def test_two_streams_at_once(kge, L):
    """Calls on two streams, each with a workspace of its own, give what each gives alone; the workspace's content does not matter."""
    a = setup("bf16", 128, 4, 1, 64, [1500, 900], [1, 1], seed=21)
    b = setup("bf16", 128, 16, 2, 16, [700, 100, 650], [1, 90, 1], seed=22)
    want = [attend(kge, s) for s in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    state = []
    for s in (a, b):
        state.append([s["q"].cuda(), s["cache"].tensor(), torch.from_numpy(s["table"]).cuda(), torch.tensor(s["lens"], **I32), torch.from_numpy(s["qsl"]).cuda(),
                      torch.zeros(kge.lib().kge_attn_kv4_workspace_bytes(s["H"], s["KV"], 128), dtype=torch.uint8, device="cuda")])
    outs = [torch.zeros_like(w) for w in want]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (q, data, table, lens, qsl, ws), out, st in zip((a, b), state, outs, streams):
            call(kge, "kge_paged_attn_kv4", out, q, q.shape[1], data, table, table.shape[1], lens, qsl, len(s["lens"]), q.shape[0], int(np.diff(s["qsl"]).max()),
                 max(s["lens"]), s["H"], s["KV"], 128, s["bs"], 128 ** -0.5, 0, 0, ws, ws.numel(), stream=st)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_maps_of_any_number_of_requests(kge, L):
    """What a launch asks of shared memory on the way to its limit: the number of requests goes up in a process of its own, so that no larger
    launch has come before."""
    body = """
import sys
sys.path[:0] = {path!r}
import numpy as np, torch
import kv4_oracle as ko
from kge_loader import load
from test_kv4_gpu import run_maps
for B in (2442, 2443, 2444, 2450, 2457, 2458, 8192):
    new = [1 + b % 3 for b in range(B)]
    a = (np.arange(2 * B, dtype=np.int32).reshape(B, 2), [b % 17 for b in range(B)], new, list(range(5 * B, 6 * B)), 3, sum(new) - 5, 16)
    got, want = run_maps(load(), *a), ko.maps(*a)
    assert (got[0] == want[0]).all() and got[1:] == tuple(want[1:]), B
print("all right")
"""
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", body.format(path=[os.path.dirname(here), here])], capture_output=True, text=True, timeout=300)
    assert "all right" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
