"""Calls of the 4-bit cache that are refused before anything is launched, and the layout's arithmetic."""
import re
import os

import numpy as np
import pytest
import torch

import kv4_oracle as ko

P = 1 << 20          # an aligned address that nothing reads


def refused(kge, rc, words):
    assert rc < 0 and re.search(words, kge.lib().kge_last_error().decode()), (rc, kge.lib().kge_last_error())


@pytest.mark.parametrize("f16", ["", "_f16"])
@pytest.mark.parametrize("change,words", [
    (dict(q_out=None), "null"), (dict(cache=None), "null"), (dict(qkv=None), "null"), (dict(slots=None), "null"), (dict(pos=None), "without positions"),
    (dict(hd=96), "head_dim"), (dict(bs=8), "power of two from 16"), (dict(bs=48), "power of two from 16"), (dict(H=0), "H=0"), (dict(KV=0), "KV=0"),
    (dict(stride=4 * 64 - 8), "apart"), (dict(stride=4 * 64 + 4), "apart"), (dict(q_out=P + 8), "aligned"), (dict(cache=P + 4), "aligned"), (dict(qkv=P + 2), "aligned"),
    (dict(cs=P + 8), "aligned"), (dict(H=1 << 20, stride=1 << 26), "heads of")])
def test_write_refusals(kge, f16, change, words):
    a = dict(q_out=P, stride=256, cache=P, qkv=P, cs=P, pos=P, slots=P, T=3, H=4, KV=2, hd=64, bs=16) | change
    refused(kge, getattr(kge.lib(), "kge_rope_kv4write" + f16)(*a.values(), None), words)


@pytest.mark.parametrize("f16", ["", "_f16"])
@pytest.mark.parametrize("change,words", [
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(cache=None), "null"), (dict(slots=None), "null"), (dict(KV=0), "KV=0"), (dict(hd=32), "head_dim"),
    (dict(bs=24), "power of two"), (dict(k=P + 8), "aligned"), (dict(cache=P + 8), "aligned")])
def test_read_refusals(kge, f16, change, words):
    a = dict(k=P, v=P, cache=P, slots=P, T=3, KV=2, hd=64, bs=16) | change
    refused(kge, getattr(kge.lib(), "kge_kv4_read" + f16)(*a.values(), None), words)


@pytest.mark.parametrize("f16", ["", "_f16"])
@pytest.mark.parametrize("change,words", [
    (dict(out=None), "null"), (dict(q=None), "null"), (dict(cache=None), "null"), (dict(table=None), "null"), (dict(lens=None), "null"), (dict(qsl=None), "null"),
    (dict(H=6, KV=4), "multiple"), (dict(H=512, KV=2, stride=512 * 64), "128 times"), (dict(hd=80), "head_dim"), (dict(bs=8), "block_size"), (dict(bs=8192), "block_size"),
    (dict(bs=40), "block_size"), (dict(stride=4 * 64 - 8), "q_stride"), (dict(stride=260), "q_stride"), (dict(out=P + 8), "aligned"), (dict(ws=P + 4), "aligned"),
    (dict(window=-1), "window"), (dict(first=-2), "window"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=-0.5), "scale"),
    (dict(maxq=0), "must be >= 1"), (dict(maxc=0), "must be >= 1"), (dict(mb=0), "must be >= 1"), (dict(mb=1 << 28), "blocks of"), (dict(B=70000), "65535"),
    (dict(ws=None), "workspace"), (dict(nws=1000), "workspace"), (dict(maxq=3, B=1, nws=1000), "workspace"),      # (before prompts are launched)
    (dict(mb=(1 << 26) + 1), "tokens a request"), (dict(scale=2e38), "scale")])
def test_attention_refusals(kge, f16, change, words):
    a = dict(out=P, q=P, stride=256, cache=P, table=P, mb=4, lens=P, qsl=P, B=3, T=3, maxq=1, maxc=50, H=4, KV=2, hd=64, bs=16, scale=0.125, window=0, first=0, ws=P,
             nws=1 << 30) | change
    refused(kge, getattr(kge.lib(), "kge_paged_attn_kv4" + f16)(*a.values(), None), words)


@pytest.mark.parametrize("change,words", [
    (dict(table=None), "null"), (dict(cached=None), "null"), (dict(free=None), "null"), (dict(first=None), "null"), (dict(bs=24), "power of two"), (dict(B=8193), "8192"),
    (dict(T=-1), "rows"), (dict(nfree=-1), "free"), (dict(mb=0), "blocks"), (dict(mb=1 << 28), "blocks")])
def test_maps_refusals(kge, change, words):
    a = dict(table=P, mb=4, lens=P, qsl=P, pos=P, slots=P, counts=P, cached=P, new=P, free=P, nfree=9, first=P, B=3, T=8, bs=16) | change
    refused(kge, kge.lib().kge_step_maps(*a.values(), None), words)


def test_sizes_beyond_32_bits_are_refused(kge):
    """Products and sums of sizes that an int does not hold, the ones that come out small again among them."""
    L = kge.lib()
    for H, KV, stride in ((3, 2 ** 31 - 1, 256), (1, 2 ** 30, 256), (2 ** 25 + 1, 1, 128), (2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 8)):
        refused(kge, L.kge_rope_kv4write(P, stride, P, P, P, P, P, 3, H, KV, 128, 16, None), "heads of|apart")
    for H, KV, stride in ((2 ** 25, 2 ** 25, 8), (2 ** 24, 2 ** 24, 2 ** 31 - 8), (2 ** 25 + 1, 2 ** 25 + 1, 256)):
        refused(kge, L.kge_paged_attn_kv4(P, P, stride, P, P, 4, P, P, 3, 3, 1, 50, H, KV, 128, 16, 0.125, 0, 0, P, 1 << 30, None), "q_stride")
    refused(kge, L.kge_step_maps(P, 4, P, P, P, P, P, P, P, P, 9, P, 3, 2 ** 31 - 1, 16, None), "rows")
    refused(kge, L.kge_kv4_read(P, P, P, P, 2 ** 31 - 1, 2 ** 31 - 1, 128, 16, None), "in one call")
    for sizes in ((2 ** 40, 2 ** 20, 128, 64), (2 ** 62, 1, 64, 16), (2 ** 33, 2 ** 31 - 1, 128, 2 ** 30)):
        assert L.kge_kv4_cache_bytes(*sizes) < 0 and b"bytes" in L.kge_last_error()


def test_calls_without_rows_do_nothing(kge):
    L = kge.lib()
    assert L.kge_rope_kv4write(P, 256, P, P, P, P, P, 0, 4, 2, 64, 16, None) == 0
    assert L.kge_kv4_read(P, P, P, P, 0, 2, 64, 16, None) == 0
    assert L.kge_paged_attn_kv4(P, P, 256, P, P, 4, P, P, 0, 0, 1, 50, 4, 2, 64, 16, 0.125, 0, 0, None, 0, None) == 0


def test_sizes(kge):
    L = kge.lib()
    assert L.kge_kv4_cache_bytes(10, 8, 128, 64) == 10 * 8 * 64 * 136
    assert L.kge_kv4_cache_bytes(1 << 22, 8, 128, 64) == (1 << 22) * 8 * 64 * 136          # beyond 32 bits
    for bad in ((-1, 8, 128, 64), (1, 0, 128, 64), (1, 8, 96, 64), (1, 8, 128, 8), (1, 8, 128, 48)):
        assert L.kge_kv4_cache_bytes(*bad) < 0
    assert L.kge_attn_kv4_workspace_bytes(32, 8, 128) > 0
    assert L.kge_attn_kv4_workspace_bytes(128, 8, 128) > L.kge_attn_kv4_workspace_bytes(32, 8, 128)
    assert L.kge_attn_kv4_workspace_bytes(40, 2, 128) == 0 and L.kge_attn_kv4_workspace_bytes(5, 2, 128) < 0


def test_the_layouts_arithmetic_is_the_oracles():
    """key_row, key_token and value_word of csrc/kv4.cuh, evaluated here."""
    src = open(os.path.join(os.path.dirname(__file__), "..", "kubernetes-gpu-cluster_b200", "csrc", "kv4.cuh")).read()
    body = {n: re.search(n + r"\(.*?\) \{ return (.*?); \}", src).group(1) for n in ("key_row", "key_token")}
    for tok in range(16):
        row = eval(body["key_row"], {"token": tok})
        assert ko.KEY_ROWS[row] == tok and eval(body["key_token"], {"row": row}) == tok
    assert "hd == 128 ? j ^ ((token & 2) << 2) : j" in src


@pytest.mark.parametrize("dtype,hd", [("bf16", 128), ("fp16", 64)])
def test_the_oracles_two_ways_agree(dtype, hd):
    """put() and put_all(), get() and parts(), attention() and attention_terms()."""
    dt, g = ko.DT[dtype], torch.Generator().manual_seed(3)
    a, b = (ko.Cache(4, 2, hd, 32, dt, fill=0xA5) for _ in range(2))
    slots = torch.randperm(128, generator=g)[:90].tolist()
    k, v = (torch.randn(90, 2, hd, generator=g).to(dt) for _ in range(2))
    k[5, 1, 3], v[7, 0, 2], v[9] = float("nan"), float("inf"), 2.5
    a.put(k, v, slots)
    b.put_all(k, v, slots)
    assert (a.data == b.data).all()
    k[5, 1, 3], v[7, 0, 2] = 1, 1
    a.put(k, v, slots)
    for whole, (code, s, low) in zip(a.get(slots, 1), a.parts(slots, 1)):
        assert torch.equal(whole, low + s * code) and code.min() >= 0 and code.max() <= 15
    c = ko.Cache(4, 2, hd, 32, dt)
    c.put_all(k, v, list(range(90)))
    table = np.array([[0, 1], [2, 1]], dtype=np.int32)
    q = torch.randn(30, 6, hd, generator=g).to(dt)
    for window, first in ((0, 0), (9, 4)):
        want = ko.attention(c, q, table, [60, 20], np.array([0, 25, 30]), 6, 0.1, window, first)[0]
        got = ko.attention_terms(c, q, table, [60, 20], np.array([0, 25, 30]), 6, 0.1, window, first)[0]
        assert (got - want).abs().max() < 1e-12
