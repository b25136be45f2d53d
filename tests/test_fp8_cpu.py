"""Calls of the 8-bit block products that are refused before anything is launched."""
import re

import pytest

P = 1 << 20          # an aligned address that nothing reads


def refused(kge, rc, words):
    assert rc < 0 and re.search(words, kge.lib().kge_last_error().decode()), (rc, kge.lib().kge_last_error())


@pytest.mark.parametrize("f16", ["", "_f16"])
@pytest.mark.parametrize("change,words", [
    (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(x=None), "null"), (dict(K=0), "multiple of 16"), (dict(K=24), "multiple of 16"), (dict(K=-16), "multiple of 16"),
    (dict(xst=120), "apart"), (dict(xst=132), "apart"), (dict(sst=2), "scales_stride"), (dict(codes=P + 8), "aligned"), (dict(x=P + 8), "aligned"), (dict(scales=P + 2), "aligned"),
    (dict(T=2 ** 31 - 1, K=2 ** 20, xst=2 ** 20, sst=2 ** 31 - 1), "in one call")])
def test_row_refusals(kge, f16, change, words):
    a = dict(codes=P, scales=P, sst=3, x=P, xst=128, rows=None, T=3, K=128) | change
    refused(kge, getattr(kge.lib(), "kge_fp8_quant" + f16)(*a.values(), None), words)


@pytest.mark.parametrize("f16", ["", "_f16"])
@pytest.mark.parametrize("change,words", [
    (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(w=None), "null"), (dict(E=0), "matrices"), (dict(N=0), "matrices"),
    (dict(E=2 ** 31 - 1, N=2 ** 31 - 1), "in one call"), (dict(K=8), "multiple of 16"), (dict(codes=P + 4), "aligned"), (dict(w=P + 4), "aligned")])
def test_weight_refusals(kge, f16, change, words):
    a = dict(codes=P, scales=P, w=P, E=2, N=100, K=128) | change
    refused(kge, getattr(kge.lib(), "kge_fp8_quant_weight" + f16)(*a.values(), None), words)


COMMON = [(dict(x=None), "null"), (dict(xs=None), "null"), (dict(w=None), "null"), (dict(ws=None), "null"), (dict(K=0), "multiple of 16"), (dict(K=200), "multiple of 16"),
          (dict(T=-1), "not negative"), (dict(N=0), "not negative"), (dict(xst=2), "apart"), (dict(x=P + 8), "aligned"), (dict(w=P + 8), "aligned"), (dict(xs=P + 2), "aligned"),
          (dict(work=None), "workspace"), (dict(nwork=1000), "workspace"), (dict(work=P + 4), "workspace"), (dict(N=2 ** 31 - 128), "weight rows")]


@pytest.mark.parametrize("f16", ["", "_f16"])
@pytest.mark.parametrize("change,words", COMMON + [(dict(y=None), "null"), (dict(y=P + 1), "aligned"), (dict(bias=P + 1), "aligned")])
def test_product_refusals(kge, f16, change, words):
    a = dict(y=P, x=P, xs=P, xst=3, w=P, ws=P, bias=None, T=3, N=128, K=256, work=P, nwork=1 << 30) | change
    refused(kge, getattr(kge.lib(), "kge_gemm_fp8" + f16)(*a.values(), None), words)


@pytest.mark.parametrize("f16", ["", "_f16"])
@pytest.mark.parametrize("change,words", COMMON + [(dict(y=None), "null"), (dict(off=None), "null"), (dict(E=0), "groups"), (dict(E=1025), "groups"), (dict(off=P + 2), "aligned"),
                                                   (dict(E=1024, N=2 ** 21), "weight rows")])
def test_grouped_refusals(kge, f16, change, words):
    a = dict(y=P, x=P, xs=P, xst=3, w=P, ws=P, off=P, E=2, T=3, N=128, K=256, work=P, nwork=1 << 30) | change
    refused(kge, getattr(kge.lib(), "kge_gemm_fp8_grouped" + f16)(*a.values(), None), words)


@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("change,words", COMMON + [(dict(codes=None), "null"), (dict(scales=None), "null"), (dict(sst=2), "apart"), (dict(N=192), "multiple of 128"),
                                                   (dict(codes=P + 8), "aligned"), (dict(scales=P + 1), "aligned"), (dict(N=2 ** 30), "weight rows")])
def test_gated_refusals(kge, grouped, change, words):
    a = dict(codes=P, scales=P, sst=3, x=P, xs=P, xst=3, w=P, ws=P, off=P, E=2, T=3, N=128, K=256, work=P, nwork=1 << 30) | change
    if grouped:
        refused(kge, kge.lib().kge_gemm_fp8_grouped_silu_gate(*a.values(), None), words)
        refused(kge, kge.lib().kge_gemm_fp8_grouped_silu_gate(*(dict(a, off=None)).values(), None), "null")
    else:
        refused(kge, kge.lib().kge_gemm_fp8_silu_gate(*[v for k, v in a.items() if k not in ("off", "E")], None), words)


@pytest.mark.parametrize("f16", ["", "_f16"])
@pytest.mark.parametrize("change,words", [(dict(rows=P + 2), "aligned"), (dict(K=2 ** 31 - 16, xst=2 ** 31 - 8), "in one call")])
def test_row_refusals_of_indexes_and_long_rows(kge, f16, change, words):
    a = dict(codes=P, scales=P, sst=3, x=P, xst=128, rows=None, T=3, K=128) | change
    refused(kge, getattr(kge.lib(), "kge_fp8_quant" + f16)(*a.values(), None), words)


def test_calls_without_rows_do_nothing(kge):
    L = kge.lib()
    assert L.kge_fp8_quant(P, P, 3, P, 128, None, 0, 128, None) == 0
    assert L.kge_gemm_fp8(P, P, P, 3, P, P, None, 0, 128, 256, None, 0, None) == 0
    assert L.kge_gemm_fp8_silu_gate(P, P, 3, P, P, 3, P, P, 0, 128, 256, None, 0, None) == 0
    assert L.kge_gemm_fp8_grouped(P, P, P, 3, P, P, P, 2, 0, 128, 256, None, 0, None) == 0
    assert L.kge_gemm_fp8_grouped_silu_gate(P, P, 3, P, P, 3, P, P, P, 2, 0, 128, 256, None, 0, None) == 0


def test_workspace_sizes(kge):
    L = kge.lib()
    assert L.kge_gemm_fp8_workspace_bytes(0) == 0 and L.kge_gemm_fp8_workspace_bytes(-5) == 0
    sizes = [L.kge_gemm_fp8_workspace_bytes(t) for t in (1, 32, 33, 64, 128, 129, 8192, 2 ** 31 - 1)]
    assert sizes == sorted(sizes) and sizes[0] == sizes[1] and sizes[4] == sizes[-1] <= 64 << 20


@pytest.mark.parametrize("f16", ["", "_f16"])
@pytest.mark.parametrize("E,N,K", [(2 ** 30, 2 ** 31 - 100, 2 ** 18), (2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 16), (2 ** 24, 2 ** 31 - 128, 2 ** 24)])
def test_matrices_whose_steps_64_bits_do_not_count(kge, f16, E, N, K):
    refused(kge, getattr(kge.lib(), "kge_fp8_quant_weight" + f16)(P, P, P, E, N, K, None), "in one call")


@pytest.mark.parametrize("f16", ["", "_f16"])
@pytest.mark.parametrize("grouped", [False, True])
def test_products_whose_tiles_64_bits_do_not_count(kge, f16, grouped):
    T = N = 2 ** 31 - 257
    args = [P, P, P, 2 ** 31 - 1, P, P, P] + ([1] if grouped else []) + [T, N, 2 ** 31 - 16, P, 1 << 30, None]
    refused(kge, getattr(kge.lib(), "kge_gemm_fp8" + ("_grouped" if grouped else "") + f16)(*args), "in one call")
    if not f16:
        f = 2 ** 30 - 256
        args = [P, P, 2 ** 31 - 1, P, P, 2 ** 31 - 1, P, P] + ([P, 1] if grouped else []) + [T, f, 2 ** 31 - 16, P, 1 << 30, None]
        refused(kge, getattr(kge.lib(), "kge_gemm_fp8" + ("_grouped" if grouped else "") + "_silu_gate")(*args), "in one call")
